// Attention over a paged KV4 cache (kv4.cuh) for many requests in one call: for each row and query head
//   out = sum over the row's cells c of p_c V[c],  p = softmax(scale q . K[c]),  times sigmoid(gate) when given.
// Row i of the m rows of a request that holds n cells sees its first n - m + i + 1 cells.
//
// What bounds it: the cells, read once.  144 bytes a 256-wide head and plane against eight query rows of a group, so the
// tensor-core work of a decode step is small (at 196 608 cells of 2 heads under 16 query heads: 113 MB, 17 us at the
// measured copy rate, against 6.4 GFLOP with the split operands) and what has to be kept small is the number of
// instructions that turn nibbles into operands.  Those decide the formulation:
//
//   Products are mma.sync m16n8k16 with the CACHE as the 16-row operand and the queries as the 8-column one, both
//   products transposed: S^T [cell][query] = K q^T, O^T [dim][query] = V^T p^T.  A group of eight query heads fills the
//   columns exactly, and the cells never leave registers between shared memory and the product.  (tcgen05.mma needs
//   128 rows and its operands in shared or tensor memory: every widened cell would be written back, 4 bytes for each
//   byte read, to use a sixteenth of the unit.)
//   K: ldmatrix hands a thread eight codes of a cell in one register; a nibble under a fixed exponent, less a constant,
//   is code - 8 in FP16, two to an instruction.  A group's sum is multiplied by its d in F32.
//   V: ldmatrix.trans hands a thread four codes of each of two cells.  Here d varies along the sum, so the operand is
//   (code - 8) d, one product more, exact in FP16 by the format.  A warp owns one group of 32 dims, whose d it needs.
//   Queries and probabilities are split into two FP16 parts (the rounded value and its rounded residual), which keeps
//   what an F32 product would: errors against 64 bits are those of an F32 evaluation.  Queries are scaled by a power of
//   two per row so that their largest lies in [2^13, 2^14), probabilities by 2^14, which keeps both parts above FP16's
//   subnormals where it matters.  The tensor core truncates its F32 sums, so no sum runs long there: scores are joined
//   per group of 32 dims and outputs per tile in rounded F32 (sums run through all tiles in the tensor core were four
//   times further from 64 bits).  Softmax statistics are F32.
//
// Work split: a unit is a tile of 128 cells (256 of narrow heads) of one (request, KV head, block of query columns), an
// item, or an item's start: its queries, first copies and last sums cost about what a tile does, and a line of tiles alone
// left the pieces with most items behind.  With none, one and two units a start: 64 requests of up to 8192 cells 68.4, 64.1 and
// 64.0 us, 40 of up to 5000 with 32 heads over 8 of 128 51.3, 44.0 and 46.1, 13 of up to five rows 57.0, 54.1 and 55.5.  What it
// costs: a lone request whose tiles divide evenly among the CTAs gives some of them one more (18 944 cells 11.9, 14.8 and 14.9).
// The units of all requests form one line that is cut into equal pieces, one for each resident CTA, wherever the requests'
// borders fall: one long request and many ragged ones both fill the machine, from lengths only the device knows.  A piece
// that holds all tiles of an item writes its rows itself; otherwise it leaves its sums, maximum and accumulators in the
// workspace and a second launch folds an item's pieces in their order.  Where a table lists few cells and there are few items, an
// item's tiles go to a cluster of CTAs instead, which join their parts through shared memory (share_of).  Results do not
// depend on timing.
//
// A CTA is eight warps.  Scores: a warp takes 16 cells (32) for eight columns.  Maxima cross the warps through shared memory,
// probabilities go there in the order of the second product's fragments, and there a warp takes 32 dims of all cells.
// Scores run a tile ahead of outputs, so one barrier a tile is enough: two K stages and three V stages, which every
// thread fills for two tiles ahead with its share of 16-byte asynchronous copies, and each thread's wait for its own
// copies before the barrier makes them everybody's (two V stages, and one tile ahead, for units of 16 columns).  Nothing
// else waits.  (Tensor-map copies, a page each, were tried first: a page's four copies are issued one after another, by
// one warp that the seven others then wait for, or that costs them registers as a ninth: 18 warps an SM put five on a
// scheduler.  The change took 61 us to 50 at 196 608 cells.)
//
// Measured on a B200, graph replays over caches larger than L2: one request of 196 608 cells, 16 heads over 2 of 256:
// 44 us, 113 MB at 2.6 TB/s; 40 requests of up to 5000 cells, 32 heads over 8 of 128: 44 us; 64 of up to 8192, 32 over 8 of 64:
// 77 us; 8 requests of up to 300 cells: 7.6 us, latency.  A warp issues some 790 instructions a tile, and issue slots are in
// use 55 to 63 % of the time, logic 35 to 43, tensor 16 to 38: no unit is at its limit, what is waited for is mostly results of the
// warp's own last instructions (1.1 to 2.4 warps an issue) with four warps a scheduler to hide them.  Cells that lie in L2 give
// the same time.
#include <atomic>
#include <type_traits>

#include "bulk_pipe.cuh"
#include "kv4.cuh"

namespace fnb {
namespace {

constexpr int kMaxReq = 2048;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr int kStart = 1;                        // units that an item's start counts
constexpr int kMaxShare = 8;                     // CTAs that share an item in the clustered form, at most
constexpr float kPShift = 14.0f;                 // a row's weights are held so that the largest is 2^14 (from 2^24 on, 1 to 2^14)

// ---- geometry -------------------------------------------------------------------------------------------------------
// HD: head_dim.  NT: blocks of eight query columns a unit serves (1, or 2 at 256); 0: four columns, whose large and small
// parts fill one block (columns 0 .. 3 and 4 .. 7), so that one product does for both and the two halves of its result
// are added at the end of the scores and of the item.
template <int HD, int NT0>
struct geo {
    static constexpr bool kPacked = NT0 == 0;
    static constexpr int NT = kPacked ? 1 : NT0, kParts = kPacked ? 1 : 2;   // words of a fragment: both parts, or either
    static constexpr int kGroups = HD / 32;                     // scales of a cell; also 32-dim groups of the output
    // cells of a tile: what a tile costs whatever its cells (the barrier, the walk, addresses) is the same for narrow heads
    static constexpr int kTile = NT == 1 && HD < 256 ? 256 : 128, kSets = kTile / 128, kSlabs = kTile / 16;
    static constexpr int kCols = kPacked ? 4 : 8 * NT;
    static constexpr int kWarps = 8, kThreads = kWarps * 32;
    static constexpr int kCellGroups = 8 / kGroups;             // warps that share a dim group (and columns) split the cells
    static constexpr int kCodeBytes = kTile * HD / 2, kScaleBytes = kTile * kGroups * 2;
    static constexpr int kUnitBytes = kCodeBytes + kScaleBytes;
    static constexpr int kCtas = 2;                             // resident on an SM (registers, shared memory)
    // V is put out a tile behind K, so a third stage lets its copies begin a tile earlier; two where the memory is short
    static constexpr int kVStages = NT == 1 ? 3 : 2, kStages = 2 + kVStages;   // K's stages, then V's
    static constexpr uint32_t kSwz = HD == 256 ? 7u : HD == 128 ? 3u : 1u;
    // shared memory
    static constexpr int ring = 0;
    static constexpr int prob = ring + kStages * kUnitBytes;    // uint4 (uint2) [2][kSlabs][NT][32]
    static constexpr int qfrag = prob + 2 * kSlabs * NT * kParts * 256;   // uint4 [NT][kGroups][kParts][32]
    static constexpr int kQueryBytes = NT * kGroups * kParts * 512;
    static constexpr int wmax = qfrag + kQueryBytes;    // float [2][kWarps][kCols]; and the queries' [kGroups][kCols]
    static constexpr int lsum = wmax + 2 * 8 * kCols * 4;       // float [kWarps][kCols]
    static constexpr int corr = lsum + 8 * kCols * 4;           // float [2][kCols]
    static constexpr int mfin = corr + 2 * kCols * 4;           // float [kCols]
    // float4: the other cell groups' accumulators.  Of 128-wide heads they fit where the queries were: those are read up to
    // the item's last scores, and the next item's are written behind a barrier of its own.
    static constexpr int kRedBytes = (kCellGroups - 1) * kGroups * NT * 1024, tail = mfin + kCols * 4;
    static constexpr bool kRedOnQueries = kRedBytes <= kQueryBytes;
    static constexpr int red = kRedOnQueries ? qfrag : tail;
    static constexpr int scan = tail + (kRedOnQueries ? 0 : kRedBytes);  // int64 [kWarps]: sums; the piece's start
    static constexpr int total = scan + (kWarps + 4) * 8 + 1024;          // + slack to align the base to 1024 bytes
    static_assert(total * kCtas + 1024 * kCtas <= 233472, "shared memory of an SM");
};

struct paged_params {
    const float *q, *gate;
    const uint8_t *k_cache, *v_cache;
    const uint16_t *k_scale, *v_scale;
    const int32_t *table, *n_cells, *row_start;
    float * out;
    float *ws_acc, *ws_ml;
    int32_t * ws_head;  // [grid][8]: what the fold has to do at the start of each piece (fold_head)
    uint32_t * err;
    int64_t cache_slots;
    int cells_max;      // what a table row can list
    int rows, n_req, table_stride, n_pages, page_shift, n_q, n_kv, group;
    float scale_log2;
    uint32_t e1024, e64;  // FP16 exponents, twice each (code_low, code_high)
    // n / group = n group_mul >> group_shift for n < 2^31: group_mul = floor(2^(31 + l) / group) + 1 with 2^l >= group is off by
    // at most group / 2^(31 + l) of 1 / group, so the product by less than 1 / group
    uint32_t group_mul, group_shift;
    bool whole;           // pieces begin where items do
    int share_shift;      // log2 of the CTAs that share an item
};

// ---- small pieces -----------------------------------------------------------------------------------------------------
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same on a sum that starts at zero
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// two F32 values as FP16 pairs: the rounded values and the rounded residuals
__device__ __forceinline__ void split2(float x, float y, uint32_t & hi, uint32_t & lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_u32(h);
    lo = h2_u32(__floats2half2_rn(__fsub_rn(x, f.x), __fsub_rn(y, f.y)));
}
// code - 8 of the codes at bits 0 .. 3, or 4 .. 7, of each half: under the exponent of 1024, or of 64, a nibble there adds
// its code exactly.  (Every nibble moved to bits 6 .. 9 would want one constant, but a shift each: the logic unit runs at
// half the rate of the other.  The bare nibble is the FP16 subnormal code x 2^-24, exact too, and would need no
// subtraction; but the tensor core aligns products by their operands' exponents, and such sums lost six bits.)  The
// exponents come as kernel arguments: of two literals, mask and exponent, each would cost an instruction.
__device__ __forceinline__ uint32_t code_low(uint32_t w, uint32_t e1024) {
    return h2_u32(__hadd2(u32_h2((w & 0x000f000fu) | e1024), u32_h2(0xe408e408u)));  // - 1032
}
__device__ __forceinline__ uint32_t code_high(uint32_t w, uint32_t e64) {
    return h2_u32(__hadd2(u32_h2((w & 0x00f000f0u) | e64), u32_h2(0xd480d480u)));    // - 72
}
__device__ __forceinline__ uint32_t times(uint32_t c, __half2 d) { return h2_u32(__hmul2(u32_h2(c), d)); }
// infinities and NaN as 0
__device__ __forceinline__ __half2 numbers_only(__half2 d) {
    const uint32_t v = h2_u32(d);
    return u32_h2(((v & 0x7c00u) == 0x7c00u ? 0u : v & 0xffffu) | ((v & 0x7c000000u) == 0x7c000000u ? 0u : v & 0xffff0000u));
}
// 2^x; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// BYTES from global to shared memory behind the thread's back, or as many zeros
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void * src, bool some) {
    if constexpr (BYTES == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16 : 0) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(some ? BYTES : 0), "n"(BYTES) : "memory");
    }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// clusters: all threads of all CTAs arrive and wait; this address in another CTA's shared memory; loads from there
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_of(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}

// A request as every thread that walks the units sees it.
struct request {
    int n, m, row0;      // cells, rows, first row
    int tiles, blocks;   // of cells, of query columns
};
template <class G>
__device__ __forceinline__ request load_request(const paged_params & p, int r, bool report) {
    request x;
    int n = __ldg(p.n_cells + r);
    x.row0 = p.row_start != nullptr ? __ldg(p.row_start + r) : r;
    int end = p.row_start != nullptr ? __ldg(p.row_start + r + 1) : r + 1;
    if (report && p.err != nullptr && (n < 0 || n > p.cells_max || x.row0 < 0 || end < x.row0 || end > p.rows)) {
        atomicOr(p.err, FNB_ERR_PAGES);
    }
    n = n < 0 ? 0 : n > p.cells_max ? p.cells_max : n;
    x.row0 = x.row0 < 0 ? 0 : x.row0;
    end = end > p.rows ? p.rows : end;
    x.n = n, x.m = end > x.row0 ? end - x.row0 : 0;
    x.tiles = n > 0 ? (n + G::kTile - 1) / G::kTile : 1;  // a request without cells still has rows to write
    x.blocks = int((int64_t(x.m) * p.group + G::kCols - 1) / G::kCols);
    return x;
}
template <bool ITEMS>
__device__ __forceinline__ int64_t units_of(const paged_params & p, const request & x) {  // or its items
    return int64_t(p.n_kv) * x.blocks * (ITEMS ? 1 : x.tiles + kStart);
}

// the walk over a piece of the line: request, KV head, column block, tile
template <class G>
struct cursor {
    int r, h, blk, tile;
    request x;
    // unit `offset` of the request: an item is its start, kStart units below 0 here, and then its tiles
    __device__ __forceinline__ void at(const paged_params & p, int request_index, uint32_t offset) {
        r = request_index;
        x = load_request<G>(p, r, false);
        const uint32_t item = offset / uint32_t(x.tiles + kStart);
        tile = int(offset - item * uint32_t(x.tiles + kStart)) - kStart;
        h = int(item / uint32_t(x.blocks));
        blk = int(item - uint32_t(h) * uint32_t(x.blocks));
    }
    // CTA `rank` of those that share an item, the request's item-th: where its tiles begin, and their number
    __device__ __forceinline__ int at_share(const paged_params & p, int request_index, uint32_t item, int rank) {
        r = request_index;
        x = load_request<G>(p, r, false);
        h = int(item / uint32_t(x.blocks));
        blk = int(item - uint32_t(h) * uint32_t(x.blocks));
        tile = int(int64_t(x.tiles) * rank >> p.share_shift);
        return int(int64_t(x.tiles) * (rank + 1) >> p.share_shift) - tile;
    }
    __device__ __forceinline__ void next_item(const paged_params & p) {
        tile = 0;
        if (++blk < x.blocks) return;
        blk = 0;
        if (++h < p.n_kv) return;
        h = 0;
        do {
            if (++r >= p.n_req) return;
            x = load_request<G>(p, r, false);
        } while (x.m == 0);
    }
};

// the line's cut into `grid` pieces: the first `more` of them hold one unit more than the others
struct pieces {
    uint32_t each, more;
    __device__ __forceinline__ pieces(uint32_t total, uint32_t grid) : each(total / grid), more(total - total / grid * grid) {}
    __device__ __forceinline__ uint32_t start(uint32_t i) const { return i * each + min(i, more); }
    __device__ __forceinline__ uint32_t holder(uint32_t u) const {  // of a unit that exists
        const uint32_t fat = more * (each + 1);
        return u < fat ? u / (each + 1) : more + (u - fat) / each;
    }
};

// What the fold does at the start of a piece: nothing, or join the pieces `from` .. `to` of the item that was cut there
// (only the first cut of an item says so).
struct __align__(16) fold_head {
    int32_t fold, from, to, h, blk, row0, m, unused;  // ..; head and column block of the item, its request's rows
};

// ---- the copies -------------------------------------------------------------------------------------------------------
// Step s of a piece brings tile s's K and tile s - kLag's V.  A warp copies sixteen rows, which lie in one page: one page
// id a warp and tile, fetched a step ahead, and addresses that differ by constants.  A lane copies one 16-byte chunk (a
// group's codes) of kPass rows, and one row's scales, K's (lower half-warp) or V's.  Chunk c of a row lies at c ^ (bits
// of the row), which keeps ldmatrix free of bank conflicts.  The walk runs two tiles ahead of the scores.
template <class G, int HD>
struct loader {
    static constexpr int kCh = G::kGroups, kRows = 32 / kCh, kPass = 16 / kRows, kRow = HD / 2, kScale = kCh * 2;
    static constexpr int kLag = 4 - G::kVStages, S = G::kSets;  // a tile is S sets of 128 rows, sixteen to a warp
    cursor<G> c;
    uint32_t step, last;      // steps so far; behind the piece's last tile
    int units;                // of the piece from this tile on
    uint32_t k_st, v_st;      // where the next copies go
    int32_t id[S];            // pages of the warp's rows in tile `step`
    uint32_t cell[kLag][S];   // first of its rows in the kLag tiles before `step` (the last first), counted through all heads of a plane
    int left[kLag];           // those tiles' cells from the warp's first row on
    uint32_t lane_to;         // this lane's chunk of the warp's first pass within a stage

    __device__ __forceinline__ static int warp_row() { return int(threadIdx.x >> 5) * 16; }
    __device__ __forceinline__ void fetch(const paged_params & p) {
        const int32_t * t = p.table + int64_t(c.r) * p.table_stride;
#pragma unroll
        for (int q = 0; q < S; ++q) {
            const int at = c.tile * G::kTile + q * 128 + warp_row();
            id[q] = at < c.x.n ? __ldg(t + (at >> p.page_shift)) : 0;
        }
    }
    __device__ __forceinline__ void start(const paged_params & p, const cursor<G> & from, int n, uint32_t ring) {
        c = from, step = 0, units = n, last = n > 0 ? 0xffffff00u : 0u, k_st = ring, v_st = ring + 2 * G::kUnitBytes;
#pragma unroll
        for (int i = 0; i < kLag; ++i) {
            left[i] = 0;
#pragma unroll
            for (int q = 0; q < S; ++q) cell[i][q] = 0;
        }
        fetch(p);
        const uint32_t lane = threadIdx.x & 31, row = uint32_t(warp_row()) + lane / kCh;
        lane_to = row * kRow + (((lane % kCh) ^ ((row * kRow >> 7) & G::kSwz)) << 4);
    }
    // `some` (at most sixteen count) of the rows at cell `first` into set q of the stage at `st`
    template <bool ALL>
    __device__ __forceinline__ void rows(const uint8_t * plane, uint32_t first, int some, uint32_t st, int q) const {
        const uint32_t lane = threadIdx.x & 31;
        const uint8_t * src = plane + uint64_t(first) * kRow + lane * 16;
        const uint32_t to = st + lane_to + q * 128 * kRow;
        // a 256-wide cell: four rows a pass, so every second pass has the other half of the eight row patterns
#pragma unroll
        for (int i = 0; i < kPass; ++i) {
            copy_async<16>((to + i * kRows * kRow) ^ (kRows == 4 && (i & 1) ? 64u : 0u), src + i * kRows * kRow, ALL || int(lane / kCh) + i * kRows < some);
        }
    }
    // scales: the lower half-warp K's, the upper V's
    template <bool ALL>
    __device__ __forceinline__ void scales(const paged_params & p, uint32_t k_cell, uint32_t v_cell, int k_some, int v_some, int q) const {
        const uint32_t lane = threadIdx.x & 31;
        const bool lower = lane < 16;
        const uint32_t at = (lower ? k_cell : v_cell) + (lane & 15);
        copy_async<kScale>((lower ? k_st : v_st) + G::kCodeBytes + uint32_t(q * 128 + warp_row() + (lane & 15)) * kScale,
                           (lower ? p.k_scale : p.v_scale) + uint64_t(at) * kCh, ALL || int(lane & 15) < (lower ? k_some : v_some));
    }
    __device__ __forceinline__ void next(const paged_params & p, uint32_t ring) {
        if (step >= last + kLag) return;
        const bool k_too = step < last, v_too = step >= uint32_t(kLag);
        const int base = c.tile * G::kTile + warp_row(), k_left = c.x.n - base, v_left = left[kLag - 1];
        const uint32_t head = uint32_t(c.h) * uint32_t(p.cache_slots), mask = (1u << p.page_shift) - 1;
        uint32_t k_cell[S];
        bool known = true;
#pragma unroll
        for (int q = 0; q < S; ++q) {
            known = known && uint32_t(id[q]) < uint32_t(p.n_pages);
            k_cell[q] = head + (uint32_t(id[q]) << p.page_shift) + (uint32_t(base + q * 128) & mask);
        }
        if (k_too && v_too && known && min(k_left, v_left) >= (S - 1) * 128 + 16) {
#pragma unroll
            for (int q = 0; q < S; ++q) {
                rows<true>(p.v_cache, cell[kLag - 1][q], 16, v_st, q);
                rows<true>(p.k_cache, k_cell[q], 16, k_st, q);
                scales<true>(p, k_cell[q], cell[kLag - 1][q], 16, 16, q);
            }
        } else {
            if (k_too && !known) {
                if ((threadIdx.x & 31) == 0 && p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
#pragma unroll
                for (int q = 0; q < S; ++q) {
                    if (uint32_t(id[q]) >= uint32_t(p.n_pages)) k_cell[q] = head + (uint32_t(base + q * 128) & mask);
                }
            }
            const int k_all = k_too ? k_left : 0, v_all = v_too ? v_left : 0;
#pragma unroll
            for (int q = 0; q < S; ++q) {
                if (v_too) rows<false>(p.v_cache, cell[kLag - 1][q], v_all - q * 128, v_st, q);
                if (k_too) rows<false>(p.k_cache, k_cell[q], k_all - q * 128, k_st, q);
                if ((threadIdx.x & 31) < 16 ? k_too : v_too) scales<false>(p, k_cell[q], cell[kLag - 1][q], k_all - q * 128, v_all - q * 128, q);
            }
        }
        copies_commit();
#pragma unroll
        for (int i = kLag - 1; i > 0; --i) {
            left[i] = left[i - 1];
#pragma unroll
            for (int q = 0; q < S; ++q) cell[i][q] = cell[i - 1][q];
        }
        left[0] = k_left;
#pragma unroll
        for (int q = 0; q < S; ++q) cell[0][q] = k_cell[q];
        ++step;
        if (k_too) {
            --units;
            if (++c.tile >= c.x.tiles) units -= kStart;
            if (units > 0) {
                if (c.tile >= c.x.tiles) c.next_item(p);
                fetch(p);
            } else {
                last = step;
            }
        }
        k_st = step & 1 ? ring + G::kUnitBytes : ring;
        if (v_too) v_st = v_st == ring + (G::kStages - 1) * G::kUnitBytes ? ring + 2 * G::kUnitBytes : v_st + G::kUnitBytes;
    }
};

// ---- the kernel -------------------------------------------------------------------------------------------------------
// SHARED: clusters of two to eight CTAs, each cluster an item at a time and each CTA an even share of its tiles; shares are
// joined through the CTAs' shared memory, in the order of the tiles, and there is no second launch.
template <int HD, int NT0, bool SHARED>
__global__ void __launch_bounds__(geo<HD, NT0>::kThreads, geo<HD, NT0>::kCtas)
attend_paged_kernel(const __grid_constant__ paged_params p) {
    using G = geo<HD, NT0>;
    constexpr int NB = G::kGroups, NT = G::NT, kParts = G::kParts;
    constexpr bool kPacked = G::kPacked;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (rounding the pointer itself would make every access a generic one)
    int64_t * s_scan = reinterpret_cast<int64_t *>(smem + G::scan);
    volatile uint32_t * s_start = reinterpret_cast<volatile uint32_t *>(s_scan + G::kWarps);  // the piece's first request, its unit there
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

    pdl_launch_dependents();
    pdl_wait();

    // where this CTA's piece starts: sums of the requests' units, formed by every CTA for itself
    const int per = (p.n_req + G::kThreads - 1) / G::kThreads;
    int64_t mine = 0;
    for (int j = 0; j < per; ++j) {
        const int r = tid * per + j;
        if (r < p.n_req) mine += units_of<SHARED>(p, load_request<G>(p, r, blockIdx.x == 0));
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(kFull, upto, o);
        if (lane >= o) upto += up;
    }
    if (lane == 31) s_scan[wid] = upto;
    __syncthreads();
    int64_t sum = 0;
#pragma unroll
    for (int w = 0; w < G::kWarps; ++w) {
        if (w < wid) upto += s_scan[w];
        sum += s_scan[w];
    }
    if (sum > INT32_MAX) {  // the same in every CTA
        if (blockIdx.x == 0 && tid == 0 && p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
        sum = 0;
    }
    const uint32_t total = uint32_t(sum);
    const pieces cut(total, gridDim.x);
    uint32_t u0 = cut.start(blockIdx.x), u1 = cut.start(blockIdx.x + 1);
    auto find = [&](uint32_t u, int slot) {  // one thread: the request that holds unit u, and the unit's place in it
        if (u < total && upto > int64_t(u) && upto - mine <= int64_t(u)) {
            int64_t base = upto - mine;
            for (int j = 0; j < per; ++j) {
                const int64_t units = units_of<SHARED>(p, load_request<G>(p, tid * per + j, false));
                if (base + units > int64_t(u)) {
                    s_start[slot] = uint32_t(tid * per + j);
                    s_start[slot + 1] = u - uint32_t(base);
                    break;
                }
                base += units;
            }
        }
    };
    [[maybe_unused]] const int rank = int(blockIdx.x) & ((1 << p.share_shift) - 1);   // in its cluster
    [[maybe_unused]] uint32_t shared_item = blockIdx.x >> p.share_shift;
    if constexpr (SHARED) u0 = shared_item;
    find(u0, 0);
    if (!SHARED && p.whole) find(u1, 2);
    __syncthreads();
    if constexpr (SHARED) {
        if (shared_item >= total) return;   // the whole cluster
        u0 = 0, u1 = 1;
    }
    if (!SHARED && p.whole && u0 < u1) {
        cursor<G> at;
        at.at(p, int(s_start[0]), s_start[1]);
        u0 -= uint32_t(at.tile + kStart);
        if (u1 < total) {
            at.at(p, int(s_start[2]), s_start[3]);
            u1 -= uint32_t(at.tile + kStart);
        }
    }
    cursor<G> c;
    if (!SHARED && u0 < u1) {
        c.at(p, int(s_start[0]), s_start[1]);
        if (p.whole) c.tile = -kStart;
        if (c.tile < 0) u0 += uint32_t(-c.tile), c.tile = 0;   // nothing to do there
    }
    if (u0 >= u1) {
        if (tid == 0 && p.ws_head != nullptr) {
            reinterpret_cast<fold_head *>(p.ws_head + int64_t(blockIdx.x) * 8)->fold = 0;
        }
        return;
    }
    if constexpr (SHARED) {
        u1 = uint32_t(c.at_share(p, int(s_start[0]), s_start[1], rank));
    }
    const uint32_t ring = smem_u32(smem) + G::ring;
    loader<G, HD> load;
    load.start(p, c, int(u1 - u0), ring);
    if (!SHARED && tid == G::kThreads - 1 && p.ws_head != nullptr) {
        fold_head f = {0, 0, 0, c.h, c.blk, c.x.row0, c.x.m, 0};
        if (c.tile != 0) {
            const uint32_t first = u0 - uint32_t(c.tile);          // the item's first unit
            f.from = int(cut.holder(first)), f.to = int(cut.holder(first + uint32_t(c.x.tiles) - 1));
            f.fold = int(blockIdx.x) == f.from + 1;                // a cut piece is never empty, so neither is the next
        }
        *reinterpret_cast<fold_head *>(p.ws_head + int64_t(blockIdx.x) * 8) = f;
    }

    const int g = lane >> 2, t = lane & 3;
    const int t2 = kPacked ? 2 * (t & 1) : 2 * t;                    // of a block's columns, this lane's first in a product's result
    constexpr int SL = G::kSets;                                     // scores: a warp's slabs of 16 cells, wid SL on
    const int dg = wid % NB, cg = wid / NB;                          // outputs: dim group, cell group
    constexpr int kSlabs = G::kSlabs / G::kCellGroups;                       // slabs of a cell group
    float * s_wmax = reinterpret_cast<float *>(smem + G::wmax);
    float * s_lsum = reinterpret_cast<float *>(smem + G::lsum);
    float * s_corr = reinterpret_cast<float *>(smem + G::corr);
    float * s_mfin = reinterpret_cast<float *>(smem + G::mfin);
    using frag = std::conditional_t<kPacked, uint2, uint4>;          // probabilities of a slab, a lane's
    frag * s_prob = reinterpret_cast<frag *>(smem + G::prob);
    uint4 * s_q = reinterpret_cast<uint4 *>(smem + G::qfrag);
    // ldmatrix: a lane's row of a tile and its 16-byte chunk there, which the loader has xored with bits of the row
    // (the same for every sixteenth row, so all addresses of a lane differ by constants)
    const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8, lhalf = lane >> 4;
    const uint32_t swz = (uint32_t(lrow) * (HD / 2) >> 7) & G::kSwz;
    const uint32_t k_off = uint32_t(wid * SL * 16 + lrow) * (HD / 2) + ((uint32_t(lhalf) ^ swz) << 4);               // groups 0, 1
    const uint32_t v_off = uint32_t(cg * kSlabs * 16 + lhalf * 16 + lrow) * (HD / 2) + ((uint32_t(dg) ^ swz) << 4);  // slabs 0, 1

    uint32_t k_at = G::ring, v_at = G::ring + 2 * G::kUnitBytes;  // stages of the next tile scored, of the next tile put out
    uint32_t u = u0;
    while (SHARED || u < u1) {
        const int tile_first = c.tile;
        const int n_tiles = int(min(uint32_t(c.x.tiles - c.tile), u1 - u));
        const bool whole = tile_first == 0 && n_tiles == c.x.tiles;      // (a share may have no tiles)
        const int col0 = c.blk * G::kCols;
        auto row_of_col = [&](int col) { return int(uint64_t(uint32_t(col0 + col)) * p.group_mul >> p.group_shift); };  // / p.group

        const int n_blocks = min(NT, (c.x.m * p.group - col0 + 7) / 8);   // column blocks with a live column
        // Queries, split, in the order of the fragments: lane (g, t) has dims 8 t + {0, 4}, {1, 5}, {2, 6}, {3, 7} of a group
        // of column 8 x + g, which are nibbles 0 .. 3 of the two halves of a cell's word.  A (column block, group) at a time
        // a warp; the rows' maxima and then the fragments cross the warps.
        auto load8 = [&](int b, int x, float4 (&v)[2]) {
            const int col = kPacked ? g & 3 : x * 8 + g, i = row_of_col(col);
            const float * src = p.q + (int64_t(c.x.row0 + i) * p.n_q + c.h * p.group + (col0 + col - i * p.group)) * HD + 32 * b + 8 * t;
            const bool on = i < c.x.m;
            v[0] = on ? __ldg(reinterpret_cast<const float4 *>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[1] = on ? __ldg(reinterpret_cast<const float4 *>(src + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
        };
        auto powers = [&](float top, float & up, float & down) {  // the power of two that takes top into [2^13, 2^14), its inverse
            int e = int(__float_as_uint(top) >> 23);
            e = e < 14 ? 14 : e > 254 ? 254 : e;
            up = __uint_as_float(uint32_t(267 - e) << 23), down = __uint_as_float(uint32_t(e - 13) << 23);
        };
        auto top_of = [&](int col) {
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) top = fmaxf(top, s_wmax[b * G::kCols + col]);
            return top;
        };
        constexpr int kPairs = NB * NT;
        float4 first[2];
        if (wid < kPairs) load8(wid % NB, wid / NB, first);
        if (load.step == 0) load.next(p, ring);              // the piece's first copies, while the queries arrive
#pragma unroll
        for (int k = 0; k * G::kWarps < kPairs; ++k) {
            const int pair = wid + k * G::kWarps, b = pair % NB, x = pair / NB;
            if (pair >= kPairs) break;
            float4 v[2] = {first[0], first[1]};
            if (k > 0) load8(b, x, v);
            float top = fmaxf(fmaxf(fmaxf(fabsf(v[0].x), fabsf(v[0].y)), fmaxf(fabsf(v[0].z), fabsf(v[0].w))),
                              fmaxf(fmaxf(fabsf(v[1].x), fabsf(v[1].y)), fmaxf(fabsf(v[1].z), fabsf(v[1].w))));
            top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
            top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
            if (t == 0) s_wmax[b * G::kCols + (kPacked ? g & 3 : x * 8 + g)] = top;
        }
        if (load.step == 1) load.next(p, ring);
        named_barrier<1>(G::kThreads);
#pragma unroll
        for (int k = 0; k * G::kWarps < kPairs; ++k) {
            const int pair = wid + k * G::kWarps, b = pair % NB, x = pair / NB;
            if (pair >= kPairs) break;
            float4 v[2] = {first[0], first[1]};
            if (k > 0) load8(b, x, v);                       // again, from L1
            float up, down;
            powers(top_of(kPacked ? g & 3 : x * 8 + g), up, down);
            uint4 hi, lo;
            split2(__fmul_rn(v[0].x, up), __fmul_rn(v[1].x, up), hi.x, lo.x);
            split2(__fmul_rn(v[0].y, up), __fmul_rn(v[1].y, up), hi.y, lo.y);
            split2(__fmul_rn(v[0].z, up), __fmul_rn(v[1].z, up), hi.z, lo.z);
            split2(__fmul_rn(v[0].w, up), __fmul_rn(v[1].w, up), hi.w, lo.w);
            if constexpr (kPacked) {
                s_q[b * 32 + lane] = g < 4 ? hi : lo;
            } else {
                s_q[(x * NB + b) * 64 + lane] = hi, s_q[(x * NB + b) * 64 + 32 + lane] = lo;
            }
        }
        // columns 8 x + t2 + z: the factor of their scores, the cells they see; running maxima, this warp's sums
        float sc[NT][2], mx[NT][2], ls[NT][2];
        int lim[NT][2];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const int col = x * 8 + t2 + z, r = row_of_col(col);
                float up, down;
                powers(top_of(col), up, down);
                sc[x][z] = fmaxf(p.scale_log2 * down, 0x1p-126f);
                lim[x][z] = r < c.x.m ? c.x.n - c.x.m + r + 1 : 0;
                mx[x][z] = -INFINITY, ls[x][z] = 0.0f;
            }
        }
        const int lim_min = c.x.n - c.x.m + row_of_col(0) + 1;   // cells every live row of the block sees
        copies_wait<1>();                                        // K of the piece's first tile
        named_barrier<1>(G::kThreads);

        float sv[SL][NT][4];
        float acc[NT][2][4];  // column block x
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[x][y][z] = 0.0f;
            }
        }

        // scores of tile `it` of the item into sv, their maxima to the other warps
        auto scores = [&](int it) {
            const int base = (tile_first + it) * G::kTile;
            const uint8_t * kt = smem + k_at;
            const uint32_t k_addr = smem_u32(smem) + k_at + k_off;
            k_at = k_at == G::ring ? G::ring + G::kUnitBytes : G::ring;
            uint32_t dk[SL][2][NB / 2];
#pragma unroll
            for (int s = 0; s < SL; ++s) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const uint8_t * at = kt + G::kCodeBytes + ((wid * SL + s) * 16 + g + 8 * z) * (NB * 2);
                    if constexpr (NB == 8) {
                        *reinterpret_cast<uint4 *>(dk[s][z]) = *reinterpret_cast<const uint4 *>(at);
                    } else if constexpr (NB == 4) {
                        *reinterpret_cast<uint2 *>(dk[s][z]) = *reinterpret_cast<const uint2 *>(at);
                    } else {
                        *reinterpret_cast<uint32_t *>(dk[s][z]) = *reinterpret_cast<const uint32_t *>(at);
                    }
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) sv[s][x][0] = sv[s][x][1] = sv[s][x][2] = sv[s][x][3] = 0.0f;
            }
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                uint32_t ka[SL][2][8];  // two groups' operands: nibbles 0 and 1, then 2 and 3
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    uint32_t w[4];
                    ldm4(w, (k_addr + s * 16 * (HD / 2)) ^ uint32_t(b << 4));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t w0 = w[2 * j], w1 = w[2 * j + 1], y0 = w0 >> 8, y1 = w1 >> 8;
                        ka[s][j][0] = code_low(w0, p.e1024), ka[s][j][1] = code_low(w1, p.e1024);
                        ka[s][j][2] = code_high(w0, p.e64), ka[s][j][3] = code_high(w1, p.e64);
                        ka[s][j][4] = code_low(y0, p.e1024), ka[s][j][5] = code_low(y1, p.e1024);
                        ka[s][j][6] = code_high(y0, p.e64), ka[s][j][7] = code_high(y1, p.e64);
                    }
                }
#pragma unroll
                for (int x = 0; x < NT; ++x) {
                    if (NT > 1 && x >= n_blocks) break;
                    uint4 hi[2], lo[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) hi[j] = s_q[(x * NB + b + j) * kParts * 32 + lane];
#pragma unroll
                    for (int j = 0; j < 2; ++j) if (!kPacked) lo[j] = s_q[(x * NB + b + j) * 64 + 32 + lane];
#pragma unroll
                    for (int s = 0; s < SL; ++s) {
                        // two groups side by side, so that their sums' chains overlap; the small parts first
                        float part[2][4];
                        if constexpr (kPacked) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) mma16816_first(part[j], ka[s][j][0], ka[s][j][1], ka[s][j][2], ka[s][j][3], hi[j].x, hi[j].y);
                        } else {
#pragma unroll
                            for (int j = 0; j < 2; ++j) mma16816_first(part[j], ka[s][j][0], ka[s][j][1], ka[s][j][2], ka[s][j][3], lo[j].x, lo[j].y);
#pragma unroll
                            for (int j = 0; j < 2; ++j) mma16816(part[j], ka[s][j][4], ka[s][j][5], ka[s][j][6], ka[s][j][7], lo[j].z, lo[j].w);
#pragma unroll
                            for (int j = 0; j < 2; ++j) mma16816(part[j], ka[s][j][0], ka[s][j][1], ka[s][j][2], ka[s][j][3], hi[j].x, hi[j].y);
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j) mma16816(part[j], ka[s][j][4], ka[s][j][5], ka[s][j][6], ka[s][j][7], hi[j].z, hi[j].w);
                        const float2 f0 = __half22float2(u32_h2(dk[s][0][b / 2])), f1 = __half22float2(u32_h2(dk[s][1][b / 2]));
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float a = j ? f0.y : f0.x, c = j ? f1.y : f1.x;
                            sv[s][x][0] = fmaf(a, part[j][0], sv[s][x][0]), sv[s][x][1] = fmaf(a, part[j][1], sv[s][x][1]);
                            sv[s][x][2] = fmaf(c, part[j][2], sv[s][x][2]), sv[s][x][3] = fmaf(c, part[j][3], sv[s][x][3]);
                        }
                    }
                }
            }
            if constexpr (kPacked) {  // the large parts' sums and the small parts'
#pragma unroll
                for (int s = 0; s < SL; ++s) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) sv[s][0][z] += __shfl_xor_sync(kFull, sv[s][0][z], 2);
                }
            }
            if (base + G::kTile > lim_min) {
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    const int cell = base + (wid * SL + s) * 16 + g;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        if (cell >= lim[x][0]) sv[s][x][0] = -INFINITY;
                        if (cell >= lim[x][1]) sv[s][x][1] = -INFINITY;
                        if (cell + 8 >= lim[x][0]) sv[s][x][2] = -INFINITY;
                        if (cell + 8 >= lim[x][1]) sv[s][x][3] = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                if (NT > 1 && x >= n_blocks) break;
                float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                for (int s = 0; s < SL; ++s) t0 = fmaxf(t0, fmaxf(sv[s][x][0], sv[s][x][2])), t1 = fmaxf(t1, fmaxf(sv[s][x][1], sv[s][x][3]));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) t0 = fmaxf(t0, __shfl_xor_sync(kFull, t0, o)), t1 = fmaxf(t1, __shfl_xor_sync(kFull, t1, o));
                if (g == 0) *reinterpret_cast<float2 *>(s_wmax + ((it & 1) * 8 + wid) * G::kCols + x * 8 + t2) = make_float2(t0, t1);
            }
        };
        // probabilities of tile `it`, in the second product's fragment order; the factor its outputs rescale the sums by
        auto weights = [&](int it, float & r0, float & r1) {
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                if (NT > 1 && x >= n_blocks) break;
                // lane (g, t) takes the maxima that the g-th warp found
                float2 v = *reinterpret_cast<const float2 *>(s_wmax + ((it & 1) * 8 + g) * G::kCols + x * 8 + t2);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) v.x = fmaxf(v.x, __shfl_xor_sync(kFull, v.x, o)), v.y = fmaxf(v.y, __shfl_xor_sync(kFull, v.y, o));
                // The reference is the maximum less kPShift, rounded up: beside scores past 2^24 the shift is lost in the
                // rounding, and only upwards does no weight pass 2^kPShift.  Products are rounded here and below alike, so
                // that the cell of the maximum has exactly the maximum's.  (Two scalar operations a score: a packed product
                // and a packed sum are compiled into one FMA, rounding modes and -fmad=false notwithstanding, and an FMA leaves
                // the product unrounded: past 2^25 that gave weights of infinity, or of zero in all cells.)
                const float n0 = fmaxf(mx[x][0], __fadd_ru(__fmul_rn(v.x, sc[x][0]), -kPShift));
                const float n1 = fmaxf(mx[x][1], __fadd_ru(__fmul_rn(v.y, sc[x][1]), -kPShift));
                const float f0 = n0 == -INFINITY ? 0.0f : n0, f1 = n1 == -INFINITY ? 0.0f : n1;
                r0 = ex2(mx[x][0] - f0), r1 = ex2(mx[x][1] - f1);
                mx[x][0] = n0, mx[x][1] = n1;
                ls[x][0] *= r0, ls[x][1] *= r1;
                if (NT > 1 && wid == 0 && g == 0) *reinterpret_cast<float2 *>(s_corr + (it & 1) * G::kCols + x * 8 + 2 * t) = make_float2(r0, r1);
#pragma unroll
                for (int s = 0; s < SL; ++s) {
                    const float e0 = ex2(__fsub_rn(__fmul_rn(sv[s][x][0], sc[x][0]), f0)), e1 = ex2(__fsub_rn(__fmul_rn(sv[s][x][1], sc[x][1]), f1));
                    const float e2 = ex2(__fsub_rn(__fmul_rn(sv[s][x][2], sc[x][0]), f0)), e3 = ex2(__fsub_rn(__fmul_rn(sv[s][x][3], sc[x][1]), f1));
                    ls[x][0] += e0 + e2, ls[x][1] += e1 + e3;
                    uint32_t h0, h1, q0, q1;
                    split2(e0, e1, h0, q0);
                    split2(e2, e3, h1, q1);
                    frag & to = s_prob[(((it & 1) * G::kSlabs + wid * SL + s) * NT + x) * 32 + lane];
                    if constexpr (kPacked) {
                        to = make_uint2(transpose8x8(t < 2 ? h0 : q0), transpose8x8(t < 2 ? h1 : q1));
                    } else {
                        to = make_uint4(transpose8x8(h0), transpose8x8(h1), transpose8x8(q0), transpose8x8(q1));
                    }
                }
            }
        };
        // tile `it`'s share of the outputs
        auto outputs_of = [&](int it, float r0, float r1, auto some_masked) {
            constexpr bool masked = decltype(some_masked)::value;   // some row does not see some cell of the tile
            const int base = (tile_first + it) * G::kTile;
            [[maybe_unused]] const uint32_t v_at_here = v_at;
            const uint8_t * vt = smem + v_at;
            const uint32_t v_addr = smem_u32(smem) + v_at + v_off;
            v_at = v_at == G::ring + (G::kStages - 1) * G::kUnitBytes ? G::ring + 2 * G::kUnitBytes : v_at + G::kUnitBytes;
            const uint16_t * dv = reinterpret_cast<const uint16_t *>(vt + G::kCodeBytes) + cg * kSlabs * 16 * NB + dg;  // this warp's cells and group
            const int valid = masked ? min(G::kTile, c.x.n - base) - cg * kSlabs * 16 : kSlabs * 16;   // of its cells, those that were copied
            uint32_t bad = 0;
            if constexpr (masked) {
                // A cell that some row does not see may hold no number.  Its scale counts as 0 below, and the rows that do
                // see it get their NaN back at the end.  (Behind the request's last cell all bytes are 0.)
#pragma unroll
                for (int j = 0; j < kSlabs / 2; ++j) {
                    if ((dv[(lane + 32 * j) * NB] & 0x7c00u) == 0x7c00u) bad |= 1u << j;
                }
            }
            // the tile's sums: with one column block the small parts (of four columns every second slab) apart: shorter chains
            float part[NT][2][4], small[2][4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
#pragma unroll
                for (int x = 0; x < NT; ++x) part[x][0][z] = part[x][1][z] = 0.0f;
                small[0][z] = small[1][z] = 0.0f;
            }
#pragma unroll
            for (int sp = 0; sp < kSlabs; sp += 2) {
                if (masked && sp * 16 >= valid) break;
                uint32_t w[4];  // cells 0-7 and 8-15 of the first slab, then of the second
                ldm4t(w, v_addr + sp * 16 * (HD / 2));
                // a 256-wide cell's scales are a matrix row: transposed, lane (g, t) has group g's of cells 2 t, 2 t + 1
                [[maybe_unused]] uint32_t ds[NB == 8 ? 4 : 1];
                if constexpr (NB == 8) ldm4t(ds, smem_u32(smem) + v_at_here + G::kCodeBytes + (sp * 16 + lane) * 16);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    __half2 da, db;  // scales of cells 2 t, 2 t + 1 and of 2 t + 8, 2 t + 9 of the slab
                    if constexpr (NB == 8) {
                        da = u32_h2(__shfl_sync(kFull, ds[2 * j], dg * 4 + t)), db = u32_h2(__shfl_sync(kFull, ds[2 * j + 1], dg * 4 + t));
                    } else {
                        const uint16_t * d = dv + ((sp + j) * 16 + 2 * t) * NB;
                        da = u32_h2(uint32_t(d[0]) | (uint32_t(d[NB]) << 16)), db = u32_h2(uint32_t(d[8 * NB]) | (uint32_t(d[9 * NB]) << 16));
                    }
                    if constexpr (masked) da = numbers_only(da), db = numbers_only(db);
                    const uint32_t y0 = w[2 * j], y1 = w[2 * j + 1], z0 = y0 >> 8, z1 = y1 >> 8;
                    const uint32_t a0 = times(code_low(y0, p.e1024), da), a1 = times(code_high(y0, p.e64), da);
                    const uint32_t a2 = times(code_low(y1, p.e1024), db), a3 = times(code_high(y1, p.e64), db);
                    const uint32_t b0 = times(code_low(z0, p.e1024), da), b1 = times(code_high(z0, p.e64), da);
                    const uint32_t b2 = times(code_low(z1, p.e1024), db), b3 = times(code_high(z1, p.e64), db);
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        if (NT > 1 && x >= n_blocks) break;
                        const frag f = s_prob[(((it & 1) * G::kSlabs + cg * kSlabs + sp + j) * NT + x) * 32 + lane];
                        if constexpr (kPacked) {
                            mma16816(j ? small[0] : part[0][0], a0, a1, a2, a3, f.x, f.y);
                            mma16816(j ? small[1] : part[0][1], b0, b1, b2, b3, f.x, f.y);
                        } else {
                            float(&s0)[4] = NT == 1 ? small[0] : part[x][0];
                            float(&s1)[4] = NT == 1 ? small[1] : part[x][1];
                            mma16816(s0, a0, a1, a2, a3, f.z, f.w);
                            mma16816(s1, b0, b1, b2, b3, f.z, f.w);
                            mma16816(part[x][0], a0, a1, a2, a3, f.x, f.y);
                            mma16816(part[x][1], b0, b1, b2, b3, f.x, f.y);
                        }
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                if (NT > 1 && x >= n_blocks) break;
                float2 f = make_float2(r0, r1);
                if (NT > 1) f = *reinterpret_cast<const float2 *>(s_corr + (it & 1) * G::kCols + x * 8 + 2 * t);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
#pragma unroll
                    for (int z = 0; z < 4; ++z) {
                        const float add = NT == 1 ? part[x][y][z] + small[y][z] : part[x][y][z];
                        acc[x][y][z] = fmaf(acc[x][y][z], z & 1 ? f.y : f.x, add);
                    }
                }
            }
            if constexpr (masked) if (__any_sync(kFull, bad != 0)) {
                for (int cell = 0; cell < kSlabs * 16; ++cell) {
                    if ((__shfl_sync(kFull, bad, cell & 31) >> (cell >> 5) & 1u) == 0) continue;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            if (base + cg * kSlabs * 16 + cell >= c.x.n - c.x.m + row_of_col(x * 8 + t2 + z) + 1) continue;
#pragma unroll
                            for (int y = 0; y < 2; ++y) acc[x][y][z] = acc[x][y][z + 2] = NAN;
                        }
                    }
                }
            }
        };

        auto outputs = [&](int it, float r0, float r1) {
            if ((tile_first + it + 1) * G::kTile > lim_min) {
                outputs_of(it, r0, r1, std::true_type{});
            } else {
                outputs_of(it, r0, r1, std::false_type{});
            }
        };

        // One barrier a tile: behind it lie the tile's scores, the probabilities of the tile before and all copies begun
        // before the last barrier.  Between two barriers a warp has three pieces of work that do not wait for one another.
        if (!SHARED || n_tiles > 0) scores(0);
        float r0 = 0.0f, r1 = 0.0f;
        for (int it = 0; it < n_tiles; ++it) {
            copies_wait<0>();
            named_barrier<1>(G::kThreads);
            load.next(p, ring);  // into the stages of this tile's K and of the V before the last
            float s0, s1;
            weights(it, s0, s1);
            if (it > 0) outputs(it - 1, r0, r1);
            if (it + 1 < n_tiles) scores(it + 1);
            r0 = s0, r1 = s1;
        }
        copies_wait<0>();
        named_barrier<1>(G::kThreads);
        if (!SHARED || n_tiles > 0) outputs(n_tiles - 1, r0, r1);

        // ---- the item's end: sums across the warps, cell groups joined, rows written or left to be folded
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                ls[x][0] += __shfl_xor_sync(kFull, ls[x][0], o), ls[x][1] += __shfl_xor_sync(kFull, ls[x][1], o);
            }
            if (g == 0) {
                *reinterpret_cast<float2 *>(s_lsum + wid * G::kCols + x * 8 + t2) = make_float2(ls[x][0], ls[x][1]);
                if (wid == 0) *reinterpret_cast<float2 *>(s_mfin + x * 8 + t2) = make_float2(mx[x][0], mx[x][1]);
            }
        }
        if constexpr (kPacked) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[0][y][z] += __shfl_xor_sync(kFull, acc[0][y][z], 2);
            }
        }
        auto write_out = [&](int64_t at, float4 o, float l) {   // sums o over the weights' sum l
            const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
            o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
            if (p.gate != nullptr) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(p.gate + at));
                o.x = __fdiv_rn(o.x, 1.0f + expf(-v.x)), o.y = __fdiv_rn(o.y, 1.0f + expf(-v.y));
                o.z = __fdiv_rn(o.z, 1.0f + expf(-v.z)), o.w = __fdiv_rn(o.w, 1.0f + expf(-v.w));
            }
            *reinterpret_cast<float4 *>(p.out + at) = o;
        };
        float4 * s_red = reinterpret_cast<float4 *>(smem + G::red);
        if (cg > 0) {
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    s_red[((((cg - 1) * NB + dg) * NT + x) * 2 + y) * 32 + lane] = make_float4(acc[x][y][0], acc[x][y][1], acc[x][y][2], acc[x][y][3]);
                }
            }
        }
        named_barrier<1>(G::kThreads);
        if (cg == 0) {
#pragma unroll
            for (int o = 1; o < G::kCellGroups; ++o) {
#pragma unroll
                for (int x = 0; x < NT; ++x) {
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float4 v = s_red[((((o - 1) * NB + dg) * NT + x) * 2 + y) * 32 + lane];
                        acc[x][y][0] += v.x, acc[x][y][1] += v.y, acc[x][y][2] += v.z, acc[x][y][3] += v.w;
                    }
                }
            }
            const int64_t slot = int64_t(blockIdx.x) * 2 + (tile_first != 0 ? 0 : 1);
#pragma unroll
            for (int x = 0; x < NT; ++x) {
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    if ((NT > 1 && x >= n_blocks) || (kPacked && t >= 2)) continue;
                    const int col = x * 8 + t2 + z, i = row_of_col(col);
                    if (i >= c.x.m) continue;
                    float l = 0.0f;
#pragma unroll
                    for (int w = 0; w < 8; ++w) l += s_lsum[w * G::kCols + col];
                    float4 o = make_float4(acc[x][0][z], acc[x][0][z + 2], acc[x][1][z], acc[x][1][z + 2]);
                    if (whole) {
                        const int64_t at = (int64_t(c.x.row0 + i) * p.n_q + c.h * p.group + (col0 + col - i * p.group)) * HD + dg * 32 + 4 * g;
                        write_out(at, o, l);
                    } else if constexpr (SHARED) {   // where the tiles were
                        *reinterpret_cast<float4 *>(smem + G::ring + (col * HD + dg * 32 + 4 * g) * 4) = o;
                        if (dg == 0 && g == 0) *reinterpret_cast<float2 *>(smem + G::ring + G::kCols * HD * 4 + col * 8) = make_float2(s_mfin[col], l);
                    } else {
                        *reinterpret_cast<float4 *>(p.ws_acc + (slot * G::kCols + col) * HD + dg * 32 + 4 * g) = o;
                        if (dg == 0 && g == 0) *reinterpret_cast<float2 *>(p.ws_ml + (slot * G::kCols + col) * 2) = make_float2(s_mfin[col], l);
                    }
                }
            }
        }
        if constexpr (SHARED) {
            if (c.x.tiles > 1) {   // the same in all CTAs of the cluster
                cluster_barrier();
                const int share = 1 << p.share_shift, each = G::kCols * HD / 4 >> p.share_shift;   // vectors of the outputs a CTA joins
                for (int at = rank * each + tid; at < (rank + 1) * each; at += G::kThreads) {
                    const int col = at / (HD / 4), v = at % (HD / 4), i = row_of_col(col);
                    if (i >= c.x.m) continue;
                    float2 ml[kMaxShare];
                    float4 a[kMaxShare];
                    float top = -INFINITY;
#pragma unroll
                    for (int o = 0; o < kMaxShare; ++o) {
                        const uint32_t from = smem_of(ring, o & (share - 1));   // all loads at once: none waits for a branch
                        ml[o] = ld_cluster2(from + uint32_t(G::kCols * HD * 4 + col * 8));
                        a[o] = ld_cluster4(from + uint32_t(at * 16));
                        top = fmaxf(top, ml[o].x);
                    }
                    const float base = top == -INFINITY ? 0.0f : top;
                    float4 o4 = make_float4(0.f, 0.f, 0.f, 0.f);
                    float sum = 0.0f;
#pragma unroll
                    for (int o = 0; o < kMaxShare; ++o) {
                        if (o >= share) break;
                        const float w = ex2(ml[o].x - base);
                        sum = fmaf(ml[o].y, w, sum);
                        o4.x = fmaf(a[o].x, w, o4.x), o4.y = fmaf(a[o].y, w, o4.y), o4.z = fmaf(a[o].z, w, o4.z), o4.w = fmaf(a[o].w, w, o4.w);
                    }
                    write_out((int64_t(c.x.row0 + i) * p.n_q + c.h * p.group + (col0 + col - i * p.group)) * HD + v * 4, o4, sum);
                }
                cluster_barrier();   // nobody reads this CTA's part any more
            }
            shared_item += gridDim.x >> p.share_shift;
            if (shared_item >= total) return;
            find(shared_item, 0);
            __syncthreads();
            u = 0, u1 = uint32_t(c.at_share(p, int(s_start[0]), s_start[1], rank));
            load.start(p, c, int(u1), ring);
            k_at = G::ring, v_at = G::ring + 2 * G::kUnitBytes;
        } else {
            u += uint32_t(n_tiles + kStart);
            if (u < u1) c.next_item(p);
        }
    }
}

// ---- the fold -----------------------------------------------------------------------------------------------------------
// One column, VEC float4 vectors of dims a block, the other threads split the pieces: weights 2^(m - max), accumulators
// and sums joined in the order of the pieces.  LISTED: block k takes the k-th, (k + gridDim.x)-th .. of the cut items,
// found by listing the pieces' marks (few items, each in many pieces: few blocks an item would leave most of the machine
// idle); all weights are made first, from maxima in shared memory.  Else block k looks at piece k + 1 alone, which costs one
// load where there is nothing to fold, and as its items lie in few pieces each thread joins its own as they arrive (when it
// was added, 40 requests of up to 5000 cells, 320 items: 43.1 us against 44.9; items in ten pieces or more lost 1 to 2 us).
constexpr int kFoldThreads = 256;
constexpr int kMaxPieces = 2 * kSmCount;
template <int HD, int COLS, int VEC, bool LISTED>
__global__ void __launch_bounds__(kFoldThreads) attend_paged_fold_kernel(const __grid_constant__ paged_params p, const int pieces_all) {
    constexpr int SPLIT = kFoldThreads / VEC;
    __shared__ float4 s_acc[SPLIT][VEC];
    [[maybe_unused]] __shared__ float s_max[kFoldThreads / 32], s_sum[kFoldThreads / 32];
    [[maybe_unused]] __shared__ float s_weight[LISTED ? kMaxPieces : 1], s_part[LISTED ? kMaxPieces : 1];
    [[maybe_unused]] __shared__ fold_head s_head[LISTED ? kMaxPieces : 1];
    [[maybe_unused]] __shared__ int s_count[2 * kFoldThreads / 32];
    constexpr int JOINED = VEC < 32 ? kFoldThreads / 32 : SPLIT;   // parts left once a warp has joined its own
    [[maybe_unused]] __shared__ float2 s_ml[JOINED];
    static_assert(kMaxPieces <= 2 * kFoldThreads, "two heads a thread");
    pdl_launch_dependents();
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, col = blockIdx.y;
    pdl_wait();
    auto head_of = [&](int i) {
        const int4 * at = reinterpret_cast<const int4 *>(p.ws_head + int64_t(i) * 8);
        const int4 a = __ldcg(at), b = __ldcg(at + 1);
        return fold_head{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    };
    int cuts = int(blockIdx.x) + 1;
    if constexpr (LISTED) {
        // the cut items, in the order of the pieces: a thread two heads, listed by their rank among those that say so
        fold_head head[2];
        uint32_t some[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = tid + j * kFoldThreads;
            head[j].fold = 0;
            if (i > 0 && i < pieces_all) head[j] = head_of(i);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            some[j] = __ballot_sync(kFull, head[j].fold != 0);
            if (lane == 0) s_count[j * (kFoldThreads / 32) + wid] = __popc(some[j]);
        }
        __syncthreads();
        cuts = 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int w = 0; w < kFoldThreads / 32; ++w) {
                if (w == wid && head[j].fold != 0) s_head[cuts + __popc(some[j] & ((1u << lane) - 1))] = head[j];
                cuts += s_count[j * (kFoldThreads / 32) + w];
            }
        }
        __syncthreads();
    }
    for (int k = blockIdx.x; k < cuts; k += gridDim.x) {
        const fold_head f = LISTED ? s_head[LISTED ? k : 0] : head_of(k + 1);
        if (!LISTED && f.fold == 0) return;
        const int row = (f.blk * COLS + col) / p.group;
        if (row >= f.m) continue;
        // The pieces after the first hold the item from their start: slot 0; in the first it is the last: slot 1.
        const int n = f.to - f.from + 1;
        auto slot_of = [&](int j) { return (int64_t(f.from + j) * 2 + (j == 0 ? 1 : 0)) * COLS + col; };
        const int v = tid % VEC, part = tid / VEC;
        float a = 0.0f, s = 0.0f;   // a dim's sum and the weights', in the first VEC * 4 threads
        if constexpr (LISTED) {
            // the first pieces' accumulators are on their way before the weights are known
            auto acc_of = [&](int j) { return __ldcg(reinterpret_cast<const float4 *>(p.ws_acc + slot_of(j) * HD) + blockIdx.z * VEC + v); };
            constexpr int kAhead = 4;
            float4 ahead[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) ahead[i] = part + i * SPLIT < n ? acc_of(part + i * SPLIT) : make_float4(0.f, 0.f, 0.f, 0.f);
            float top = -INFINITY;
            for (int j = tid; j < n; j += kFoldThreads) {
                const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.ws_ml + slot_of(j) * 2));
                s_weight[j] = ml.x, s_part[j] = ml.y;
                top = fmaxf(top, ml.x);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
            if (lane == 0) s_max[wid] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kFoldThreads / 32; ++w) top = fmaxf(top, s_max[w]);
            const float base = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            for (int j = tid; j < n; j += kFoldThreads) {
                const float w = ex2(s_weight[j] - base);
                s_weight[j] = w;
                sum = fmaf(s_part[j], w, sum);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
            if (lane == 0) s_sum[wid] = sum;
            __syncthreads();
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            auto join = [&](float4 a, float w) {
                acc.x = fmaf(a.x, w, acc.x), acc.y = fmaf(a.y, w, acc.y), acc.z = fmaf(a.z, w, acc.z), acc.w = fmaf(a.w, w, acc.w);
            };
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (part + i * SPLIT < n) join(ahead[i], s_weight[part + i * SPLIT]);
            }
#pragma unroll 8
            for (int j = part + kAhead * SPLIT; j < n; j += SPLIT) join(acc_of(j), s_weight[j]);
            s_acc[part][v] = acc;
            __syncthreads();
            if (tid < VEC * 4) {
                for (int o = 0; o < min(SPLIT, n); ++o) a += reinterpret_cast<const float *>(s_acc[o])[tid];
#pragma unroll
                for (int w = 0; w < kFoldThreads / 32; ++w) s += s_sum[w];
            }
        } else {
            // a thread's pieces: maximum, sum and accumulators so far, brought to a common maximum as each is joined
            float top = -INFINITY, sum = 0.0f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            auto join = [&](float2 ml, float4 x) {
                const float t = fmaxf(top, ml.x), base = t == -INFINITY ? 0.0f : t;
                const float w0 = ex2(top - base), w1 = ex2(ml.x - base);
                top = t, sum = fmaf(ml.y, w1, sum * w0);
                acc.x = fmaf(x.x, w1, acc.x * w0), acc.y = fmaf(x.y, w1, acc.y * w0), acc.z = fmaf(x.z, w1, acc.z * w0), acc.w = fmaf(x.w, w1, acc.w * w0);
            };
            constexpr int kAhead = 4;
            for (int j = part; j < n; j += kAhead * SPLIT) {
                float2 ml[kAhead];
                float4 x[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    ml[i] = make_float2(-INFINITY, 0.0f), x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (j + i * SPLIT >= n) continue;
                    const int64_t at = slot_of(j + i * SPLIT);
                    ml[i] = __ldcg(reinterpret_cast<const float2 *>(p.ws_ml + at * 2));
                    x[i] = __ldcg(reinterpret_cast<const float4 *>(p.ws_acc + at * HD) + blockIdx.z * VEC + v);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) join(ml[i], x[i]);
            }
            if constexpr (VEC < 32) {
#pragma unroll
                for (int o = VEC; o < 32; o <<= 1) {
                    const float2 ml = make_float2(__shfl_xor_sync(kFull, top, o), __shfl_xor_sync(kFull, sum, o));
                    join(ml, make_float4(__shfl_xor_sync(kFull, acc.x, o), __shfl_xor_sync(kFull, acc.y, o), __shfl_xor_sync(kFull, acc.z, o),
                                         __shfl_xor_sync(kFull, acc.w, o)));
                }
            }
            const int joined = VEC < 32 ? wid : part;
            if (VEC >= 32 || lane < VEC) s_acc[joined][v] = acc;
            if (VEC >= 32 ? v == 0 : lane == 0) s_ml[joined] = make_float2(top, sum);
            __syncthreads();
            if (tid < VEC * 4) {
                float t = -INFINITY;
#pragma unroll
                for (int o = 0; o < JOINED; ++o) t = fmaxf(t, s_ml[o].x);
                const float base = t == -INFINITY ? 0.0f : t;
#pragma unroll
                for (int o = 0; o < JOINED; ++o) {
                    const float w = ex2(s_ml[o].x - base);
                    a = fmaf(reinterpret_cast<const float *>(s_acc[o])[tid], w, a), s = fmaf(s_ml[o].y, w, s);
                }
            }
        }
        if (tid < VEC * 4) {
            float y = s == 0.0f ? 0.0f : __fdiv_rn(a, s);
            const int64_t at = (int64_t(f.row0 + row) * p.n_q + f.h * p.group + (f.blk * COLS + col - row * p.group)) * HD + blockIdx.z * VEC * 4 + tid;
            if (p.gate != nullptr) y = __fdiv_rn(y, 1.0f + expf(-__ldg(p.gate + at)));
            p.out[at] = y;
        }
        __syncthreads();
    }
}

// ---- launch -------------------------------------------------------------------------------------------------------------
template <int HD, int NT, bool SHARED>
bool configure() {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!done[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(attend_paged_kernel<HD, NT, SHARED>, cudaFuncAttributeMaxDynamicSharedMemorySize, geo<HD, NT>::total) != cudaSuccess) {
            (void) cudaGetLastError();
            return false;
        }
        done[dev].store(true, std::memory_order_release);
    }
    return true;
}

// Column blocks of eight a unit serves, or 0.  A 256-wide head's cells are read once for sixteen columns where a request has
// that many; further columns are further passes.  (196 608 cells of 2 heads: two rows, 16 columns a head, 66 us against 75
// in two passes; eight rows, 64 columns, 215 us against 231 and 270 with units of 32 and 64 columns, whose sums leave
// registers for one CTA an SM.)  Narrow heads fare better with one block and the larger tiles it leaves room for (32
// requests of up to 4096 cells, 8 heads of 128, eight rows of four: 92 us against 97).  Up to four columns share a block
// between their large and small parts, 0 here: half the products (40 requests of up to 5000 cells, 32 heads over 8 of 128:
// 51 us against 58; 196 608 cells, 8 over 2 of 256: 36.8 against 42.7).  64-wide heads, whose tiles hold the least work next
// to what a tile costs anyway, have nothing from it (32 requests, 32 over 8: 35.5 against 33.9).
int column_blocks(const fnb_attend_paged_args * a) {
    const int64_t cols = int64_t(a->max_rows > 0 ? a->max_rows : 1) * (a->n_q_heads / a->n_kv_heads);
    if (cols <= 4 && a->head_dim >= 128) return 0;
    return a->head_dim == 256 && cols > 8 ? 2 : 1;
}
constexpr int kGrid = 2 * kSmCount;  // two CTAs an SM
// Many items of a tile or two stay whole: a CTA takes them from end to end, and there is nothing to fold.  (Cut, an item of
// three tiles has them side by side, and the fold costs less than three tiles in a row.)
constexpr int kWholeTiles = 2;
bool whole_items(const fnb_attend_paged_args * a) { return int64_t(a->max_pages) * a->page_size <= kWholeTiles * 128; }
size_t paged_workspace(const fnb_attend_paged_args * a) {
    if (whole_items(a)) return 16;  // none is used
    const int nt = column_blocks(a);
    const size_t grid = size_t(kGrid), cols = nt == 0 ? 4 : size_t(8 * nt);
    return grid * 2 * cols * (size_t(a->head_dim) + 2) * 4 + grid * 32;
}

bool paged_shape_ok(const fnb_attend_paged_args * a) {
    if (a == nullptr) return false;
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return false;
    if (a->rows < 1 || a->n_req < 1 || a->n_req > kMaxReq || a->max_pages < 1 || a->max_rows < 0) return false;
    if (a->table_stride != 0 && a->table_stride < a->max_pages) return false;
    if (a->row_start == nullptr && a->rows < a->n_req) return false;
    if (int64_t(a->rows) * a->n_q_heads > INT32_MAX) return false;
    if (a->n_q_heads < 1 || a->n_kv_heads < 1 || a->n_q_heads > 1024 || a->n_q_heads % a->n_kv_heads != 0) return false;
    if (a->page_size < 16 || a->page_size > (1 << 20) || (a->page_size & (a->page_size - 1)) != 0) return false;
    if (a->cache_slots < a->page_size || a->cache_slots > INT32_MAX || a->cache_slots % a->page_size != 0) return false;
    if (a->cache_slots * a->n_kv_heads > int64_t(UINT32_MAX)) return false;
    return true;
}

template <int HD, int NT>
int64_t expected_items(const fnb_attend_paged_args * a, const paged_params & p) {   // by max_rows, a hint: a wrong one costs time only
    constexpr int kCols = geo<HD, NT>::kCols;
    const int64_t blocks = (int64_t(a->max_rows > 0 ? a->max_rows : 1) * p.group + kCols - 1) / kCols;
    return int64_t(a->n_req) * a->n_kv_heads * blocks;
}
// The shared form: short items, few enough that each can have a cluster at once.  As many CTAs as tiles where the grid
// allows it (two for one tile), else the most that leave a CTA two tiles; items that are longer or more numerous go on the line.
// Nothing is left in memory and the second launch falls away (16 heads over 2 of 256, us, line against shared: 8 requests of up
// to 300 cells 10.5 and 7.6, 64 of up to 500 18.4 and 12.6, one of 1000 9.6 and 7.7, 16 of 2000 14.3 and 12.4; but 64 of 1000, four
// tiles a CTA, 20.5 and 22).  A lone tile gains too, against an item a CTA takes whole: the walk is shorter (one request of
// 128 cells 6.0 and 5.5, 70 of them 8.5 and 7.4).  Returns log2 of the CTAs, 0 for the line.
template <int HD, int NT>
int share_of(const paged_params & p, int64_t items) {
    const int64_t tiles = (p.cells_max + geo<HD, NT>::kTile - 1) / geo<HD, NT>::kTile;
    for (int shift = 1; shift <= 3; ++shift) {
        if (tiles <= int64_t(1) << shift && items << shift <= kGrid) return shift;
    }
    for (int shift = 3; shift >= 1; --shift) {
        if (tiles <= int64_t(2) << shift && items << shift <= kGrid) return shift;
    }
    return 0;
}

void launch_fold(void (*kernel)(paged_params, int), dim3 blocks, cudaStream_t s, const paged_params & p, int grid) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks, cfg.blockDim = dim3(kFoldThreads), cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    (void) cudaLaunchKernelEx(&cfg, kernel, p, grid);
}

template <int HD, int NT>
int32_t launch_paged(const fnb_attend_paged_args * a, paged_params & p, cudaStream_t s) {
    constexpr int kCols = geo<HD, NT>::kCols;
    const int64_t items = expected_items<HD, NT>(a, p);
    p.share_shift = share_of<HD, NT>(p, items);
    if (p.share_shift > 0) {
        if (!configure<HD, NT, true>()) return FNB_LAUNCH_FAILED;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(items < kGrid >> p.share_shift ? items : kGrid >> p.share_shift) << p.share_shift);
        cfg.blockDim = dim3(unsigned(geo<HD, NT>::kThreads));
        cfg.dynamicSmemBytes = geo<HD, NT>::total, cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = 1u << p.share_shift, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr, cfg.numAttrs = 2;
        (void) cudaLaunchKernelEx(&cfg, attend_paged_kernel<HD, NT, true>, p);
        return launch_status();
    }
    if (!configure<HD, NT, false>()) return FNB_LAUNCH_FAILED;
    const int grid = kGrid;
    const size_t cols = kCols;
    const bool fold = !p.whole;
    if (fold) {
        uint8_t * ws = static_cast<uint8_t *>(a->workspace);
        p.ws_head = reinterpret_cast<int32_t *>(ws);
        p.ws_acc = reinterpret_cast<float *>(ws + size_t(grid) * 32);
        p.ws_ml = p.ws_acc + size_t(grid) * 2 * cols * HD;
    }
    launch_pdl(attend_paged_kernel<HD, NT, false>, grid, geo<HD, NT>::kThreads, geo<HD, NT>::total, s, p);
    if (cudaPeekAtLastError() != cudaSuccess) return FNB_LAUNCH_FAILED;
    if (fold) {
        // Few items: list them, and where each may lie in 64 pieces or more, a block takes 32 dims instead of a whole head
        // (one request, 16 heads over 2 of 256, by 32 dims, by heads, unlisted: 4096 cells 11.0, 10.9 and 10.8 us, 8192 12.0,
        // 13.9 and 14.7, 196 608 43.7, 46.9 and 56.6; 20 requests of up to 4096, where the blocks are more than run at a time, 29.0,
        // 19.6 and 19.1).  Unlisted from a wave of columns on (40 requests of 32 over 8 heads of 128: 49.1 listed, 44.0).
        const int64_t outputs = items * int64_t(cols), wave = kSmCount * 8;   // columns to fold; blocks that run at a time
        if (outputs * (HD / 32) <= wave && p.cells_max >= 64 * 128) {
            launch_fold(attend_paged_fold_kernel<HD, kCols, 8, true>, dim3(unsigned(items), unsigned(cols), HD / 32), s, p, grid);
        } else if (outputs <= wave) {
            launch_fold(attend_paged_fold_kernel<HD, kCols, HD / 4, true>, dim3(unsigned(items), unsigned(cols), 1), s, p, grid);
        } else {
            launch_fold(attend_paged_fold_kernel<HD, kCols, HD / 4, false>, dim3(unsigned(grid - 1), unsigned(cols), 1), s, p, grid);
        }
    }
    return launch_status();
}
}  // namespace

template <int HD, int NT>
bool configure_both() {
    return configure<HD, NT, false>() && configure<HD, NT, true>();
}
bool attend_paged_prepare_device() {
    return configure_both<256, 0>() && configure_both<256, 1>() && configure_both<256, 2>() && configure_both<128, 0>() &&
           configure_both<128, 1>() && configure_both<64, 1>();
}

}  // namespace fnb

extern "C" size_t fnb_attend_paged_workspace_bytes(const fnb_attend_paged_args * a) {
    return fnb::paged_shape_ok(a) ? fnb::paged_workspace(a) : 0;
}

extern "C" int32_t fnb_attend_paged_kv4(const fnb_attend_paged_args * a, void * stream) {
    using namespace fnb;
    if (!paged_shape_ok(a)) return FNB_REJECTED;
    if (!ok_ptr(a->q, 16) || !ok_opt(a->gate, 16) || !ok_ptr(a->out, 16) || !ok_ptr(a->k_cache, 16) || !ok_ptr(a->v_cache, 16) ||
        !ok_ptr(a->k_scale, 16) || !ok_ptr(a->v_scale, 16)) {
        return FNB_REJECTED;
    }
    if (!ok_ptr(a->table, 4) || !ok_ptr(a->n_cells, 4) || !ok_opt(a->row_start, 4) || !ok_opt(a->err, 4)) return FNB_REJECTED;
    if (!(a->scale > 0.0f) || !(a->scale < INFINITY)) return FNB_REJECTED;
    if (!whole_items(a) && (!ok_ptr(a->workspace, 16) || a->workspace_bytes < paged_workspace(a))) return FNB_REJECTED;
    paged_params p = {};
    p.k_cache = static_cast<const uint8_t *>(a->k_cache), p.v_cache = static_cast<const uint8_t *>(a->v_cache);
    p.q = a->q, p.gate = a->gate, p.k_scale = a->k_scale, p.v_scale = a->v_scale;
    p.table = a->table, p.n_cells = a->n_cells, p.row_start = a->row_start, p.out = a->out, p.err = a->err;
    p.cache_slots = a->cache_slots, p.rows = a->rows, p.n_req = a->n_req;
    p.table_stride = a->table_stride != 0 ? a->table_stride : a->max_pages;
    const int64_t held = int64_t(a->max_pages) * a->page_size;
    p.cells_max = int(held < INT32_MAX - 256 ? held : INT32_MAX - 256);
    p.n_pages = int(a->cache_slots / a->page_size), p.page_shift = __builtin_ctz(unsigned(a->page_size));
    p.n_q = a->n_q_heads, p.n_kv = a->n_kv_heads, p.group = a->n_q_heads / a->n_kv_heads;
    p.scale_log2 = a->scale * kLog2eF;
    int l = 0;
    while ((1 << l) < p.group) ++l;
    p.group_shift = 31 + l, p.group_mul = uint32_t((uint64_t(1) << p.group_shift) / uint64_t(p.group) + 1);
    p.whole = whole_items(a);
    p.e1024 = 0x64006400u, p.e64 = 0x54005400u;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int blocks = column_blocks(a);
    switch (a->head_dim) {
        case 256: return blocks == 0 ? launch_paged<256, 0>(a, p, s) : blocks == 1 ? launch_paged<256, 1>(a, p, s) : launch_paged<256, 2>(a, p, s);
        case 128: return blocks == 0 ? launch_paged<128, 0>(a, p, s) : launch_paged<128, 1>(a, p, s);
        default: return launch_paged<64, 1>(a, p, s);
    }
}
