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
// Work split: a unit is a tile of 128 cells of one (request, KV head, block of query columns).  The units of all
// requests form one line that is cut into equal pieces, one for each resident CTA, wherever the requests' borders fall:
// one long request and many ragged ones both fill the machine, from lengths only the device knows.  A piece that holds
// all tiles of an item writes its rows itself; otherwise it leaves its sums, maximum and accumulators in the workspace
// and a second launch folds an item's pieces in their order.  Results do not depend on timing.
//
// A CTA is eight warps.  Scores: a warp takes 16 cells for eight columns, whose query fragments it keeps in registers.
// Maxima cross the warps through shared memory, probabilities go there in the order of the second product's fragments,
// and there a warp takes 32 dims of all cells.  K and V tiles take turns in a ring that warp 0 feeds: per page one
// tensor-map copy of a plane's codes, swizzled so that ldmatrix has no bank conflicts, and one bulk copy of its scales.
// The barrier between a tile's scores and its probabilities is also the proof that the tile's K stage and the V stage
// before it are no longer read, so the ring needs no barriers of its own for that, and no warp is set aside for the
// copies (a ninth warp would cost the other eight a quarter of their registers: 18 warps an SM put five on a scheduler).
#include <cuda.h>  // CUtensorMap and the type of cuTensorMapEncodeTiled (reached through cudaGetDriverEntryPoint)

#include <atomic>

#include "bulk_pipe.cuh"
#include "kv4.cuh"

namespace fnb {
namespace {

constexpr int kTileCells = 128;
constexpr int kWarpsC = 8;
constexpr int kThreadsC = kWarpsC * 32;
constexpr int kMaxReq = 2048;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr float kPShift = 14.0f;                 // probabilities are held times 2^14

// ---- geometry -------------------------------------------------------------------------------------------------------
// HD: head_dim.  NT: blocks of eight query columns a unit serves (1, 2, 4 or 8).
template <int HD, int NT>
struct geo {
    static constexpr int kGroups = HD / 32;                     // scales of a cell; also 32-dim groups of the output
    static constexpr int kCols = 8 * NT;
    static constexpr int kCellGroups = kWarpsC / kGroups;       // warps that share a dim group split the cells
    static constexpr int kCodeBytes = kTileCells * HD / 2, kScaleBytes = kTileCells * kGroups * 2;
    static constexpr int kUnitBytes = kCodeBytes + kScaleBytes;
    static constexpr int kCtas = NT <= 2 ? 2 : 1;               // resident on an SM (registers)
    static constexpr int kRing = HD == 256 ? (NT <= 2 ? 5 : 7) : (NT <= 2 ? 9 : 13);  // odd (feed_step)
    static constexpr uint32_t kSwz = HD == 256 ? 7u : HD == 128 ? 3u : 1u;
    // shared memory
    static constexpr int ring = 0;
    static constexpr int prob = ring + kRing * kUnitBytes;      // uint4 [2][8 slabs][NT][32]
    static constexpr int wmax = prob + 2 * 8 * NT * 512;        // float [2][8 warps][8]
    static constexpr int lsum = wmax + 512;                     // float [8 warps][8]
    static constexpr int corr = lsum + 256;                     // float [2][kCols]
    static constexpr int mfin = corr + 2 * kCols * 4;           // float [kCols]
    static constexpr int red = mfin + kCols * 4;                // float4: the other cell groups' accumulators
    static constexpr int bars = red + (kCellGroups - 1) * kGroups * 32 * kCols * 4;
    static constexpr int scan = bars + kRing * 8;               // int64 [8]: sums; then the start of this CTA's piece
    static constexpr int feed = scan + 12 * 8;                  // the feeder's walk
    static constexpr int total = feed + 64 + 1024;              // + slack to align the base to 1024 bytes
    static_assert(total * kCtas + 1024 * kCtas <= 233472, "shared memory of an SM");
};

struct paged_params {
    const float *q, *gate;
    const uint16_t *k_scale, *v_scale;
    const int32_t *table, *n_cells, *row_start;
    float * out;
    float *ws_acc, *ws_ml;
    int32_t * ws_head;  // [grid][8]: what the fold has to do at the start of each piece (fold_head)
    uint32_t * err;
    int64_t cache_slots;
    int cells_max;      // what a table row can list
    int rows, n_req, max_pages, n_pages, page_shift, n_q, n_kv, group;
    float scale_log2;
    uint32_t e1024, e64;  // FP16 exponents, twice each (code_low, code_high)
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
// 2^x; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tensor_g2s(void * dst, const CUtensorMap * map, int y, int z, uint64_t * bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(0), "r"(y), "r"(z), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}
// bounded; once a wait has run out, the CTA's others return at their next look and it runs to its end on what it has
__device__ __forceinline__ bool ring_wait(uint64_t * bar, uint32_t parity, volatile uint32_t * gave_up, uint32_t * err) {
    for (uint32_t i = 0; i < kPrimarySpinLimit; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63u) == 63u && *gave_up != 0) return false;
    }
    *gave_up = 1;
    if (err != nullptr) atomicOr(err, FNB_ERR_TIMEOUT);
    return false;
}

// A request as every thread that walks the units sees it.
struct request {
    int n, m, row0;      // cells, rows, first row
    int tiles, blocks;   // of cells, of query columns
};
template <int COLS>
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
    x.tiles = n > 0 ? (n + kTileCells - 1) / kTileCells : 1;  // a request without cells still has rows to write
    x.blocks = int((int64_t(x.m) * p.group + COLS - 1) / COLS);
    return x;
}
__device__ __forceinline__ int64_t units_of(const paged_params & p, const request & x) {
    return int64_t(p.n_kv) * x.blocks * x.tiles;
}

// the walk over a piece of the line: request, KV head, column block, tile
template <int COLS>
struct cursor {
    int r, h, blk, tile;
    request x;
    __device__ __forceinline__ void at(const paged_params & p, int request_index, uint32_t offset) {
        r = request_index;
        x = load_request<COLS>(p, r, false);
        const uint32_t item = offset / uint32_t(x.tiles);
        tile = int(offset - item * uint32_t(x.tiles));
        h = int(item / uint32_t(x.blocks));
        blk = int(item - uint32_t(h) * uint32_t(x.blocks));
    }
    __device__ __forceinline__ void next_item(const paged_params & p) {
        tile = 0;
        if (++blk < x.blocks) return;
        blk = 0;
        if (++h < p.n_kv) return;
        h = 0;
        do {
            if (++r >= p.n_req) return;
            x = load_request<COLS>(p, r, false);
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
struct fold_head {
    int32_t fold, from, to, r, h, blk;
};

// ---- the ring's feeder: warp 0's walk, kept in shared memory (its registers are the query fragments') ----------------
// The ring's order is K0 | K1 V0 | K2 V1 | ... | V(n - 1), the order in which stages fall free: scores run a tile ahead of
// outputs.  Step j issues K(j) from the lower half-warp and V(j - 1) from the upper one, a lane a page.
struct feeder {
    int r, h, blk, tile;
    int n, m, tiles, blocks;   // the walk's request
    uint32_t step, tiles_all;  // tiles of the piece
    int stage;                 // the next unit's
    int v_h, v_live;           // head and pages of the tile whose V is next
};
// where tile j's K and V are, of n tiles
__device__ __forceinline__ uint32_t unit_of_k(uint32_t j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ uint32_t unit_of_v(uint32_t j, uint32_t n) { return j + 1 < n ? 2 * j + 2 : 2 * n - 1; }

// One step, if there is one.  Warp 0, all lanes.  `id`: this (lower) lane's page of the K tile, fetched a step ahead;
// `slot`: this (upper) lane's first slot of the V tile.
template <int HD, int NT>
__device__ __forceinline__ void feed_step(const paged_params & p, const CUtensorMap * map_k, const CUtensorMap * map_v, feeder * f,
                                          uint8_t * smem, uint64_t * full, int32_t & slot, int32_t & id, uint64_t policy) {
    using G = geo<HD, NT>;
    const uint32_t j = f->step, n = f->tiles_all;
    if (j > n) return;
    const int lane = threadIdx.x & 31, at = lane & 15;
    const bool upper = lane >= 16;
    const int page = 1 << p.page_shift, box = page < kTileCells ? page : kTileCells;
    const int base = f->tile * kTileCells, left = f->n - base, h = f->h;
    const int k_live = j == n || left <= 0 ? 0 : min(kTileCells / box, (left + box - 1) / box);
    const int live = upper ? f->v_live : k_live;
    int stage = f->stage;
    if (upper && j > 0 && j < n) stage = stage + 1 == G::kRing ? 0 : stage + 1;
    if (!upper && at < k_live) {
        if (id < 0 || id >= p.n_pages) {
            if (p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
            id = 0;
        }
        slot = int32_t((uint32_t(id) << p.page_shift) + uint32_t((base + at * box) & (page - 1)));
    }
    uint8_t * st = smem + G::ring + stage * G::kUnitBytes;
    if (at == 0 && (upper ? j > 0 : j < n)) {
        mbar_expect_tx(&full[stage], uint32_t(live) * uint32_t(box) * (HD / 2 + G::kGroups * 2));
        mbar_arrive(&full[stage]);
    }
    __syncwarp();
    if (at < live) {
        const int head = upper ? f->v_h : h;
        tensor_g2s(st + at * box * (HD / 2), upper ? map_v : map_k, slot, head, &full[stage], policy);
        const uint16_t * scale = (upper ? p.v_scale : p.k_scale) + (int64_t(head) * p.cache_slots + slot) * G::kGroups;
        bulk_g2s(st + G::kCodeBytes + at * box * G::kGroups * 2, scale, uint32_t(box) * G::kGroups * 2, &full[stage], policy);
    }
    slot = __shfl_sync(kFull, slot, at);
    __syncwarp();
    if (lane == 0) {
        f->v_h = h, f->v_live = k_live, f->step = j + 1;
        const int next = f->stage + (j == 0 || j == n ? 1 : 2);
        f->stage = next >= G::kRing ? next - G::kRing : next;
    }
    if (j + 1 < n) {
        cursor<G::kCols> c;
        c.r = f->r, c.h = h, c.blk = f->blk, c.tile = f->tile + 1;
        c.x.n = f->n, c.x.m = f->m, c.x.tiles = f->tiles, c.x.blocks = f->blocks;
        if (c.tile >= c.x.tiles) {
            c.next_item(p);
            __syncwarp();
            if (lane == 0) {
                f->r = c.r, f->h = c.h, f->blk = c.blk;
                f->n = c.x.n, f->m = c.x.m, f->tiles = c.x.tiles, f->blocks = c.x.blocks;
            }
        }
        __syncwarp();
        if (lane == 0) f->tile = c.tile;
        const int cell = c.tile * kTileCells + at * box;
        id = !upper && at * box < kTileCells && cell < c.x.n ? __ldg(p.table + int64_t(c.r) * p.max_pages + (cell >> p.page_shift)) : -1;
    }
    __syncwarp();
}

// ---- the kernel -------------------------------------------------------------------------------------------------------
template <int HD, int NT>
__global__ void __launch_bounds__(kThreadsC, geo<HD, NT>::kCtas)
attend_paged_kernel(const paged_params p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using G = geo<HD, NT>;
    constexpr int NB = G::kGroups;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (rounding the pointer itself would make every access a generic one)
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + G::bars);
    feeder * s_feed = reinterpret_cast<feeder *>(smem + G::feed);
    int64_t * s_scan = reinterpret_cast<int64_t *>(smem + G::scan);
    volatile uint32_t * s_misc = reinterpret_cast<volatile uint32_t *>(s_scan + 8);  // [0] start request, [1] gave up, [2] start within it
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;

    pdl_launch_dependents();
    if (tid == 0) {
        for (int s = 0; s < G::kRing; ++s) {
            mbar_init(&full[s], 1);
        }
        mbar_init_fence();
        s_misc[1] = 0;
    }
    pdl_wait();

    // where this CTA's piece starts: sums of the requests' units, formed by every CTA for itself
    const int per = (p.n_req + kThreadsC - 1) / kThreadsC;
    int64_t mine = 0;
    for (int j = 0; j < per; ++j) {
        const int r = tid * per + j;
        if (r < p.n_req) mine += units_of(p, load_request<G::kCols>(p, r, blockIdx.x == 0));
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
    for (int w = 0; w < kWarpsC; ++w) {
        if (w < wid) upto += s_scan[w];
        sum += s_scan[w];
    }
    if (sum > INT32_MAX) {  // the same in every CTA
        if (blockIdx.x == 0 && tid == 0 && p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
        sum = 0;
    }
    const uint32_t total = uint32_t(sum);
    const pieces cut(total, gridDim.x);
    const uint32_t u0 = cut.start(blockIdx.x), u1 = cut.start(blockIdx.x + 1);
    if (u0 < u1 && upto > int64_t(u0) && upto - mine <= int64_t(u0)) {  // one thread
        int64_t base = upto - mine;
        for (int j = 0; j < per; ++j) {
            const int64_t units = units_of(p, load_request<G::kCols>(p, tid * per + j, false));
            if (base + units > int64_t(u0)) {
                s_misc[0] = uint32_t(tid * per + j);
                s_misc[2] = u0 - uint32_t(base);
                break;
            }
            base += units;
        }
    }
    __syncthreads();
    if (u0 >= u1) {
        if (tid == 0 && p.ws_head != nullptr) reinterpret_cast<fold_head *>(p.ws_head + int64_t(blockIdx.x) * 8)->fold = 0;
        return;
    }
    cursor<G::kCols> c;
    c.at(p, int(s_misc[0]), s_misc[2]);
    if (tid == kThreadsC - 1 && p.ws_head != nullptr) {
        fold_head f = {0, 0, 0, c.r, c.h, c.blk};
        if (c.tile != 0) {
            const uint32_t first = u0 - uint32_t(c.tile);          // the item's first unit
            f.from = int(cut.holder(first)), f.to = int(cut.holder(first + uint32_t(c.x.tiles) - 1));
            f.fold = int(blockIdx.x) == f.from + 1;                // a cut piece is never empty, so neither is the next
        }
        *reinterpret_cast<fold_head *>(p.ws_head + int64_t(blockIdx.x) * 8) = f;
    }

    // the ring is filled before anything else
    const uint64_t policy = l2_evict_first_policy();
    int32_t feed_slot = 0, feed_id = -1;  // warp 0's
    auto feed = [&]() {
        if (s_misc[1] == 0) feed_step<HD, NT>(p, &map_k, &map_v, s_feed, smem, full, feed_slot, feed_id, policy);
    };
    if (wid == 0) {
        const int page = 1 << p.page_shift, box = page < kTileCells ? page : kTileCells;
        const int at = lane & 15, cell = c.tile * kTileCells + at * box;
        feed_id = lane < 16 && at * box < kTileCells && cell < c.x.n ? __ldg(p.table + int64_t(c.r) * p.max_pages + (cell >> p.page_shift)) : -1;
        if (lane == 0) {
            s_feed->r = c.r, s_feed->h = c.h, s_feed->blk = c.blk, s_feed->tile = c.tile;
            s_feed->n = c.x.n, s_feed->m = c.x.m, s_feed->tiles = c.x.tiles, s_feed->blocks = c.x.blocks;
            s_feed->step = 0, s_feed->tiles_all = u1 - u0, s_feed->stage = 0, s_feed->v_h = 0, s_feed->v_live = 0;
        }
        __syncwarp();
        for (int k = 0; k <= G::kRing / 2; ++k) feed();
    }

    const int g = lane >> 2, t = lane & 3;
    const int nt = wid % NT, slab0 = wid / NT * NT;                  // scores: column block and first of NT slabs
    const int dg = wid % NB, cg = wid / NB;                          // outputs: dim group, cell group
    constexpr int kSlabs = 8 / G::kCellGroups;                       // slabs of a cell group
    float * s_wmax = reinterpret_cast<float *>(smem + G::wmax);
    float * s_lsum = reinterpret_cast<float *>(smem + G::lsum);
    float * s_corr = reinterpret_cast<float *>(smem + G::corr);
    float * s_mfin = reinterpret_cast<float *>(smem + G::mfin);
    uint4 * s_prob = reinterpret_cast<uint4 *>(smem + G::prob);
    // ldmatrix: a lane's row of a tile and its 16-byte chunk there, which the copy's swizzle has xored with bits of the
    // row (the same for every sixteenth row, so all addresses of a lane differ by constants)
    const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8, lhalf = lane >> 4;
    const uint32_t swz = (uint32_t(lrow) * (HD / 2) >> 7) & G::kSwz;
    const uint32_t k_off = uint32_t(slab0 * 16 + lrow) * (HD / 2) + ((uint32_t(lhalf) ^ swz) << 4);                 // groups 0, 1
    const uint32_t v_off = uint32_t(cg * kSlabs * 16 + lhalf * 16 + lrow) * (HD / 2) + ((uint32_t(dg) ^ swz) << 4);  // slabs 0, 1

    uint32_t tile_no = 0;  // tiles of the piece begun
    auto unit_ready = [&](uint32_t unit) {
        const uint32_t turn = unit / G::kRing, stage = unit - turn * G::kRing;
        (void) ring_wait(&full[stage], turn & 1u, s_misc + 1, p.err);
        return smem + G::ring + stage * G::kUnitBytes;
    };
    uint32_t u = u0;
    while (u < u1) {
        const int tile_first = c.tile;
        const int n_tiles = int(min(uint32_t(c.x.tiles - c.tile), u1 - u));
        const bool whole = tile_first == 0 && n_tiles == c.x.tiles;
        const int col0 = c.blk * G::kCols;
        auto row_of_col = [&](int col) { return (col0 + col) / p.group; };

        // queries of column 8 nt + g: this lane's eight dims of every group, in the order of the fragments
        uint32_t qf[NB][8];      // per group: n0n1 hi b0 b1, lo b0 b1; n2n3 hi, lo
        float sc0, sc1;
        int lim0, lim1;
        {
            const int col = nt * 8 + g, i = row_of_col(col);
            const bool on = i < c.x.m;
            const float * src = p.q + (int64_t(c.x.row0 + (on ? i : 0)) * p.n_q + c.h * p.group + (col0 + col) % p.group) * HD + 8 * t;
            float4 v[NB][2];
            float top = 0.0f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                v[b][0] = on ? __ldg(reinterpret_cast<const float4 *>(src + 32 * b)) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[b][1] = on ? __ldg(reinterpret_cast<const float4 *>(src + 32 * b + 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(v[b][j].x), fabsf(v[b][j].y)), fmaxf(fabsf(v[b][j].z), fabsf(v[b][j].w))));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
            top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
            int e = int(__float_as_uint(top) >> 23);
            e = e < 14 ? 14 : e > 254 ? 254 : e;
            const float up = __uint_as_float(uint32_t(267 - e) << 23), down = __uint_as_float(uint32_t(e - 13) << 23);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // dims 8 t + {0, 4}, {1, 5}, {2, 6}, {3, 7}: nibbles 0 .. 3 of the two halves of a cell's word
                split2(__fmul_rn(v[b][0].x, up), __fmul_rn(v[b][1].x, up), qf[b][0], qf[b][2]);
                split2(__fmul_rn(v[b][0].y, up), __fmul_rn(v[b][1].y, up), qf[b][1], qf[b][3]);
                split2(__fmul_rn(v[b][0].z, up), __fmul_rn(v[b][1].z, up), qf[b][4], qf[b][6]);
                split2(__fmul_rn(v[b][0].w, up), __fmul_rn(v[b][1].w, up), qf[b][5], qf[b][7]);
            }
            const float sc = fmaxf(p.scale_log2 * down, 0x1p-126f);
            sc0 = __shfl_sync(kFull, sc, 8 * t), sc1 = __shfl_sync(kFull, sc, 8 * t + 4);
            const int i0 = row_of_col(nt * 8 + 2 * t), i1 = row_of_col(nt * 8 + 2 * t + 1);
            lim0 = i0 < c.x.m ? c.x.n - c.x.m + i0 + 1 : 0, lim1 = i1 < c.x.m ? c.x.n - c.x.m + i1 + 1 : 0;
        }
        const int lim_min = c.x.n - c.x.m + row_of_col(0) + 1;   // cells every live row of the block sees

        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float sv[NT][4];
        float acc[NT][2][4];
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
            const int base = (tile_first + it) * kTileCells;
            uint8_t * kt = unit_ready(unit_of_k(tile_no + it));
            const uint32_t k_addr = smem_u32(kt) + k_off;
#pragma unroll
            for (int s = 0; s < NT; ++s) {
                const int row = (slab0 + s) * 16;
                const uint8_t * at0 = kt + G::kCodeBytes + (row + g) * (NB * 2), * at1 = at0 + 8 * NB * 2;
                sv[s][0] = sv[s][1] = sv[s][2] = sv[s][3] = 0.0f;
                uint32_t dk[2][NB / 2];
                if constexpr (NB == 8) {
                    *reinterpret_cast<uint4 *>(dk[0]) = *reinterpret_cast<const uint4 *>(at0);
                    *reinterpret_cast<uint4 *>(dk[1]) = *reinterpret_cast<const uint4 *>(at1);
                } else if constexpr (NB == 4) {
                    *reinterpret_cast<uint2 *>(dk[0]) = *reinterpret_cast<const uint2 *>(at0);
                    *reinterpret_cast<uint2 *>(dk[1]) = *reinterpret_cast<const uint2 *>(at1);
                } else {
                    *reinterpret_cast<uint32_t *>(dk[0]) = *reinterpret_cast<const uint32_t *>(at0);
                    *reinterpret_cast<uint32_t *>(dk[1]) = *reinterpret_cast<const uint32_t *>(at1);
                }
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    uint32_t w[4];
                    ldm4(w, (k_addr + s * 16 * (HD / 2)) ^ uint32_t(b << 4));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float part[4];
                        const uint32_t x0 = w[2 * j], x1 = w[2 * j + 1], y0 = x0 >> 8, y1 = x1 >> 8;
                        const uint32_t a0 = code_low(x0, p.e1024), a1 = code_low(x1, p.e1024), a2 = code_high(x0, p.e64), a3 = code_high(x1, p.e64);
                        const uint32_t e0 = code_low(y0, p.e1024), e1 = code_low(y1, p.e1024), e2 = code_high(y0, p.e64), e3 = code_high(y1, p.e64);
                        mma16816_first(part, a0, a1, a2, a3, qf[b + j][2], qf[b + j][3]);   // the small parts first
                        mma16816(part, e0, e1, e2, e3, qf[b + j][6], qf[b + j][7]);
                        mma16816(part, a0, a1, a2, a3, qf[b + j][0], qf[b + j][1]);
                        mma16816(part, e0, e1, e2, e3, qf[b + j][4], qf[b + j][5]);
                        const float2 f0 = __half22float2(u32_h2(dk[0][b / 2])), f1 = __half22float2(u32_h2(dk[1][b / 2]));
                        const float d0 = j ? f0.y : f0.x, d1 = j ? f1.y : f1.x;
                        sv[s][0] = fmaf(d0, part[0], sv[s][0]), sv[s][1] = fmaf(d0, part[1], sv[s][1]);
                        sv[s][2] = fmaf(d1, part[2], sv[s][2]), sv[s][3] = fmaf(d1, part[3], sv[s][3]);
                    }
                }
                if (base + kTileCells > lim_min) {
                    const int cell = base + row + g;
                    if (cell >= lim0) sv[s][0] = -INFINITY;
                    if (cell >= lim1) sv[s][1] = -INFINITY;
                    if (cell + 8 >= lim0) sv[s][2] = -INFINITY;
                    if (cell + 8 >= lim1) sv[s][3] = -INFINITY;
                }
            }
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int s = 0; s < NT; ++s) t0 = fmaxf(t0, fmaxf(sv[s][0], sv[s][2])), t1 = fmaxf(t1, fmaxf(sv[s][1], sv[s][3]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) t0 = fmaxf(t0, __shfl_xor_sync(kFull, t0, o)), t1 = fmaxf(t1, __shfl_xor_sync(kFull, t1, o));
            if (g == 0) *reinterpret_cast<float2 *>(s_wmax + (it & 1) * 64 + wid * 8 + 2 * t) = make_float2(t0, t1);
        };
        // probabilities of tile `it`, in the second product's fragment order; the factor its outputs rescale the sums by
        auto weights = [&](int it, float & r0, float & r1) {
            // lane (g, t) takes the maxima that the g-th of the column block's warps found
            float2 v = *reinterpret_cast<const float2 *>(s_wmax + (it & 1) * 64 + ((g % (8 / NT)) * NT + nt) * 8 + 2 * t);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) v.x = fmaxf(v.x, __shfl_xor_sync(kFull, v.x, o)), v.y = fmaxf(v.y, __shfl_xor_sync(kFull, v.y, o));
            const float n0 = fmaxf(m0, v.x * sc0), n1 = fmaxf(m1, v.y * sc1);
            const float f0 = n0 == -INFINITY ? 0.0f : n0, f1 = n1 == -INFINITY ? 0.0f : n1;
            r0 = ex2(m0 - f0), r1 = ex2(m1 - f1);
            m0 = n0, m1 = n1;
            l0 *= r0, l1 *= r1;
            if (NT > 1 && slab0 == 0 && g == 0) *reinterpret_cast<float2 *>(s_corr + (it & 1) * G::kCols + nt * 8 + 2 * t) = make_float2(r0, r1);
            const float b0 = kPShift - f0, b1 = kPShift - f1;
#pragma unroll
            for (int s = 0; s < NT; ++s) {
                const float e0 = ex2(fmaf(sv[s][0], sc0, b0)), e1 = ex2(fmaf(sv[s][1], sc1, b1));
                const float e2 = ex2(fmaf(sv[s][2], sc0, b0)), e3 = ex2(fmaf(sv[s][3], sc1, b1));
                l0 += e0 + e2, l1 += e1 + e3;
                uint32_t h0, h1, q0, q1;
                split2(e0, e1, h0, q0);
                split2(e2, e3, h1, q1);
                s_prob[(((it & 1) * 8 + slab0 + s) * NT + nt) * 32 + lane] =
                    make_uint4(transpose8x8(h0), transpose8x8(h1), transpose8x8(q0), transpose8x8(q1));
            }
        };
        // tile `it`'s share of the outputs
        auto outputs = [&](int it, float r0, float r1) {
            const int base = (tile_first + it) * kTileCells;
            const bool masked = base + kTileCells > lim_min;
            uint8_t * vt = unit_ready(unit_of_v(tile_no + it, u1 - u0));
            const uint32_t v_addr = smem_u32(vt) + v_off;
            uint16_t * dv = reinterpret_cast<uint16_t *>(vt + G::kCodeBytes) + cg * kSlabs * 16 * NB + dg;  // this warp's cells and group
            const int valid = min(kTileCells, c.x.n - base) - cg * kSlabs * 16;    // of its cells, those that were copied
            uint32_t bad = 0;
            if (masked) {
                // Behind the request's last cell lies whatever the memory held, and a cell that some row does not see may
                // hold no number: this warp's scales of such cells become 0.  (The latter are put back below, for the
                // rows that see them.)  The ring's next copy into this stage comes after them.
#pragma unroll
                for (int j = 0; j < kSlabs / 2; ++j) {
                    const int cell = lane + 32 * j;
                    const bool none = (dv[cell * NB] & 0x7c00u) == 0x7c00u;
                    if (cell < valid && none) bad |= 1u << j;
                    if (cell >= valid || none) dv[cell * NB] = 0;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
            }
            constexpr int NH = NT > 4 ? 4 : NT;                 // column blocks at a time (registers)
#pragma unroll
            for (int x0 = 0; x0 < NT; x0 += NH) {
                float part[NH][2][4], small[NH == 1 ? 2 : 1][4];
#pragma unroll
                for (int z = 0; z < 4; ++z) {
#pragma unroll
                    for (int x = 0; x < NH; ++x) part[x][0][z] = part[x][1][z] = 0.0f;
                    small[0][z] = 0.0f;
                    if (NH == 1) small[NH == 1 ? 1 : 0][z] = 0.0f;
                }
#pragma unroll
                for (int sp = 0; sp < kSlabs; sp += 2) {
                    if (sp * 16 >= valid) break;
                    uint32_t w[4];  // cells 0-7 and 8-15 of the first slab, then of the second
                    ldm4t(w, v_addr + sp * 16 * (HD / 2));
                    // a 256-wide cell's scales are a matrix row: transposed, lane (g, t) has group g's of cells 2 t, 2 t + 1
                    uint32_t ds[NB == 8 ? 4 : 1];
                    if constexpr (NB == 8) ldm4t(ds, smem_u32(vt) + G::kCodeBytes + (sp * 16 + lane) * 16);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        __half2 da, db;  // scales of cells 2 t, 2 t + 1 and of 2 t + 8, 2 t + 9 of the slab
                        if constexpr (NB == 8) {
                            da = u32_h2(__shfl_sync(kFull, ds[2 * j], dg * 4 + t)), db = u32_h2(__shfl_sync(kFull, ds[2 * j + 1], dg * 4 + t));
                        } else {
                            const uint16_t * d = dv + ((sp + j) * 16 + 2 * t) * NB;
                            da = u32_h2(uint32_t(d[0]) | (uint32_t(d[NB]) << 16)), db = u32_h2(uint32_t(d[8 * NB]) | (uint32_t(d[9 * NB]) << 16));
                        }
                        const uint32_t y0 = w[2 * j], y1 = w[2 * j + 1], z0 = y0 >> 8, z1 = y1 >> 8;
                        const uint32_t a0 = times(code_low(y0, p.e1024), da), a1 = times(code_high(y0, p.e64), da);
                        const uint32_t a2 = times(code_low(y1, p.e1024), db), a3 = times(code_high(y1, p.e64), db);
                        const uint32_t b0 = times(code_low(z0, p.e1024), da), b1 = times(code_high(z0, p.e64), da);
                        const uint32_t b2 = times(code_low(z1, p.e1024), db), b3 = times(code_high(z1, p.e64), db);
#pragma unroll
                        for (int x = 0; x < NH; ++x) {
                            const uint4 f = s_prob[(((it & 1) * 8 + cg * kSlabs + sp + j) * NT + x0 + x) * 32 + lane];
                            if constexpr (NH == 1) {
                                mma16816(small[0], a0, a1, a2, a3, f.z, f.w);
                                mma16816(small[NH == 1 ? 1 : 0], b0, b1, b2, b3, f.z, f.w);
                            } else {
                                mma16816(part[x][0], a0, a1, a2, a3, f.z, f.w);
                                mma16816(part[x][1], b0, b1, b2, b3, f.z, f.w);
                            }
                            mma16816(part[x][0], a0, a1, a2, a3, f.x, f.y);
                            mma16816(part[x][1], b0, b1, b2, b3, f.x, f.y);
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < NH; ++x) {
                    float2 f = make_float2(r0, r1);
                    if (NT > 1) f = *reinterpret_cast<const float2 *>(s_corr + (it & 1) * G::kCols + (x0 + x) * 8 + 2 * t);
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float add = NH == 1 ? part[x][y][z] + small[NH == 1 ? y : 0][z] : part[x][y][z];
                            acc[x0 + x][y][z] = fmaf(acc[x0 + x][y][z], z & 1 ? f.y : f.x, add);
                        }
                    }
                }
            }
            if (masked && __any_sync(kFull, bad != 0)) {
                for (int cell = 0; cell < kSlabs * 16; ++cell) {
                    if ((__shfl_sync(kFull, bad, cell & 31) >> (cell >> 5) & 1u) == 0) continue;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            if (base + cg * kSlabs * 16 + cell >= c.x.n - c.x.m + row_of_col(x * 8 + 2 * t + z) + 1) continue;
#pragma unroll
                            for (int y = 0; y < 2; ++y) acc[x][y][z] = acc[x][y][z + 2] = NAN;
                        }
                    }
                }
            }
        };

        // One barrier a tile: behind it lie the tile's scores and the probabilities of the tile before, and between two
        // of them a warp has three pieces of work that do not wait for one another.
        scores(0);
        float r0 = 0.0f, r1 = 0.0f;
        for (int it = 0; it < n_tiles; ++it) {
            named_barrier<1>(kThreadsC);
            if (wid == 0) {
                // no longer read: this tile's K and everything before it in the ring (the V of the tile before is behind it)
                if (tile_no + uint32_t(it) > 0) feed();
            }
            float s0, s1;
            weights(it, s0, s1);
            if (it > 0) outputs(it - 1, r0, r1);
            if (it + 1 < n_tiles) scores(it + 1);
            r0 = s0, r1 = s1;
        }
        named_barrier<1>(kThreadsC);
        outputs(n_tiles - 1, r0, r1);
        tile_no += uint32_t(n_tiles);

        // ---- the item's end: sums across the warps, cell groups joined, rows written or left to be folded
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l0 += __shfl_xor_sync(kFull, l0, o), l1 += __shfl_xor_sync(kFull, l1, o);
        if (g == 0) {
            *reinterpret_cast<float2 *>(s_lsum + wid * 8 + 2 * t) = make_float2(l0, l1);
            if (slab0 == 0) *reinterpret_cast<float2 *>(s_mfin + nt * 8 + 2 * t) = make_float2(m0, m1);
        }
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
        named_barrier<1>(kThreadsC);
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
                    const int col = x * 8 + 2 * t + z, i = row_of_col(col);
                    if (i >= c.x.m) continue;
                    float l = 0.0f;
#pragma unroll
                    for (int w = 0; w < 8 / NT; ++w) l += s_lsum[(w * NT + x) * 8 + 2 * t + z];
                    float4 o = make_float4(acc[x][0][z], acc[x][0][z + 2], acc[x][1][z], acc[x][1][z + 2]);
                    if (whole) {
                        const int64_t at = (int64_t(c.x.row0 + i) * p.n_q + c.h * p.group + (col0 + col) % p.group) * HD + dg * 32 + 4 * g;
                        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                        o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
                        if (p.gate != nullptr) {
                            const float4 v = __ldg(reinterpret_cast<const float4 *>(p.gate + at));
                            o.x = __fdiv_rn(o.x, 1.0f + expf(-v.x)), o.y = __fdiv_rn(o.y, 1.0f + expf(-v.y));
                            o.z = __fdiv_rn(o.z, 1.0f + expf(-v.z)), o.w = __fdiv_rn(o.w, 1.0f + expf(-v.w));
                        }
                        *reinterpret_cast<float4 *>(p.out + at) = o;
                    } else {
                        *reinterpret_cast<float4 *>(p.ws_acc + (slot * G::kCols + col) * HD + dg * 32 + 4 * g) = o;
                        if (dg == 0 && g == 0) *reinterpret_cast<float2 *>(p.ws_ml + (slot * G::kCols + col) * 2) = make_float2(s_mfin[col], l);
                    }
                }
            }
        }
        u += uint32_t(n_tiles);
        if (u < u1) c.next_item(p);
    }
    // after a wait that ran out: every copy has landed before the CTA's shared memory can be handed on
    if (tid == 0) {
        const uint32_t done = s_feed->step, k = done == 0 ? 0 : done > s_feed->tiles_all ? 2 * s_feed->tiles_all : 2 * done - 1;  // units issued
        for (uint32_t j = 1; j <= uint32_t(G::kRing) && j <= k; ++j) mbar_wait_landed(&full[(k - j) % G::kRing], ((k - j) / G::kRing) & 1u);
    }
}

// ---- the fold -----------------------------------------------------------------------------------------------------------
// Block (i, col): if piece i + 1 is the second of an item's, the item's pieces are folded for one column:
// weights 2^(m - max), accumulators and sums joined in the order of the pieces, eight warps taking every eighth piece.
constexpr int kFoldWarps = 8;
template <int HD, int NT>
__global__ void __launch_bounds__(kFoldWarps * 32) attend_paged_fold_kernel(const paged_params p) {
    constexpr int COLS = 8 * NT, V = HD / 128 > 0 ? HD / 128 : 1;   // float4 vectors of a lane
    constexpr int LANES = HD / 4 < 32 ? HD / 4 : 32;
    __shared__ float4 s_acc[kFoldWarps][HD / 4];
    __shared__ float s_max[kFoldWarps], s_sum[kFoldWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int col = blockIdx.y;
    const fold_head f = *reinterpret_cast<const fold_head *>(p.ws_head + int64_t(blockIdx.x + 1) * 8);
    if (f.fold == 0) return;
    const request x = load_request<COLS>(p, f.r, false);
    const int row = (f.blk * COLS + col) / p.group;
    if (row >= x.m) return;

    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    float4 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.0f;
    // the pieces after the first hold the item from their start: slot 0; in the first it is the last: slot 1
#pragma unroll 4
    for (int j = f.from + wid; j <= f.to; j += kFoldWarps) {
        const int64_t slot = int64_t(j) * 2 + (j == f.from ? 1 : 0);
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.ws_ml + (slot * COLS + col) * 2));
        float4 a[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[v] = lane < LANES ? __ldcg(reinterpret_cast<const float4 *>(p.ws_acc + (slot * COLS + col) * HD) + lane + 32 * v)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.0f : top;
        const float wo = ex2(m - base), wn = ex2(ml.x - base);
        m = top;
        l = fmaf(l, wo, ml.y * wn);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            acc[v].x = fmaf(acc[v].x, wo, a[v].x * wn), acc[v].y = fmaf(acc[v].y, wo, a[v].y * wn);
            acc[v].z = fmaf(acc[v].z, wo, a[v].z * wn), acc[v].w = fmaf(acc[v].w, wo, a[v].w * wn);
        }
    }
    if (lane < LANES) {
#pragma unroll
        for (int v = 0; v < V; ++v) s_acc[wid][lane + 32 * v] = acc[v];
    }
    if (lane == 0) s_max[wid] = m, s_sum[wid] = l;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= HD) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kFoldWarps; ++w) top = fmaxf(top, s_max[w]);
    const float base = top == -INFINITY ? 0.0f : top;
    float a = 0.0f, s = 0.0f;
#pragma unroll
    for (int w = 0; w < kFoldWarps; ++w) {
        const float k = ex2(s_max[w] - base);
        a = fmaf(reinterpret_cast<const float *>(s_acc[w])[d], k, a);
        s = fmaf(s_sum[w], k, s);
    }
    float y = s == 0.0f ? 0.0f : __fdiv_rn(a, s);
    const int64_t at = (int64_t(x.row0 + row) * p.n_q + f.h * p.group + (f.blk * COLS + col) % p.group) * HD + d;
    if (p.gate != nullptr) y = __fdiv_rn(y, 1.0f + expf(-__ldg(p.gate + at)));
    p.out[at] = y;
}

// ---- launch -------------------------------------------------------------------------------------------------------------
using encode_fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
encode_fn encode_tensor_map() {
    static const encode_fn fn = [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            (void) cudaGetLastError();
            return encode_fn(nullptr);
        }
        return reinterpret_cast<encode_fn>(f);
    }();
    return fn;
}
// a plane's codes [kv head][slot][hd / 2 bytes], 16 bits an element; the box one page (at most a tile) of one head, its
// cells' 16-byte chunks swizzled over the whole cell
bool make_map(CUtensorMap * map, const void * codes, int64_t slots, int n_kv, int hd, int box) {
    const encode_fn enc = encode_tensor_map();
    if (enc == nullptr) return false;
    const cuuint64_t dims[3] = {cuuint64_t(hd / 4), cuuint64_t(slots), cuuint64_t(n_kv)};
    const cuuint64_t strides[2] = {cuuint64_t(hd / 2), cuuint64_t(slots) * cuuint64_t(hd / 2)};
    const cuuint32_t boxes[3] = {cuuint32_t(hd / 4), cuuint32_t(box), 1u}, elem[3] = {1u, 1u, 1u};
    const CUtensorMapSwizzle swz = hd == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : hd == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void *>(codes), dims, strides, boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
               swz, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int NT>
bool configure() {
    static std::atomic<bool> done[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!done[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(attend_paged_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, geo<HD, NT>::total) != cudaSuccess) {
            (void) cudaGetLastError();
            return false;
        }
        done[dev].store(true, std::memory_order_release);
    }
    return true;
}

// Column blocks a unit serves: enough for a request of `max_rows` rows, so that its cells are read once; at most eight
// (more rows are served by further passes over the cells).
int column_blocks(const fnb_attend_paged_args * a) {
    const int64_t cols = int64_t(a->max_rows > 0 ? a->max_rows : 1) * (a->n_q_heads / a->n_kv_heads);
    return cols <= 8 ? 1 : cols <= 16 ? 2 : cols <= 32 ? 4 : 8;
}
int ctas_of(int nt) { return kSmCount * (nt <= 2 ? 2 : 1); }
bool one_tile(const fnb_attend_paged_args * a) { return int64_t(a->max_pages) * a->page_size <= kTileCells; }
size_t paged_workspace(const fnb_attend_paged_args * a) {
    if (one_tile(a)) return 16;  // no item is longer than a unit: nothing to fold
    const int nt = column_blocks(a);
    const size_t grid = size_t(ctas_of(nt)), cols = size_t(8 * nt);
    return grid * 2 * cols * (size_t(a->head_dim) + 2) * 4 + grid * 32;
}

bool paged_shape_ok(const fnb_attend_paged_args * a) {
    if (a == nullptr) return false;
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return false;
    if (a->rows < 1 || a->n_req < 1 || a->n_req > kMaxReq || a->max_pages < 1 || a->max_rows < 0) return false;
    if (a->row_start == nullptr && a->rows < a->n_req) return false;
    if (a->n_q_heads < 1 || a->n_kv_heads < 1 || a->n_q_heads > 1024 || a->n_q_heads % a->n_kv_heads != 0) return false;
    if (a->page_size < 16 || a->page_size > (1 << 20) || (a->page_size & (a->page_size - 1)) != 0) return false;
    if (a->cache_slots < a->page_size || a->cache_slots > INT32_MAX || a->cache_slots % a->page_size != 0) return false;
    return true;
}

template <int HD, int NT>
int32_t launch_paged(const fnb_attend_paged_args * a, paged_params & p, cudaStream_t s) {
    const int box = a->page_size < kTileCells ? a->page_size : kTileCells;
    CUtensorMap map_k, map_v;
    if (!make_map(&map_k, a->k_cache, a->cache_slots, a->n_kv_heads, HD, box) || !make_map(&map_v, a->v_cache, a->cache_slots, a->n_kv_heads, HD, box) ||
        !configure<HD, NT>()) {
        return FNB_LAUNCH_FAILED;
    }
    const int grid = ctas_of(NT);
    const size_t cols = 8 * NT;
    const bool fold = !one_tile(a);
    if (fold) {
        uint8_t * ws = static_cast<uint8_t *>(a->workspace);
        p.ws_head = reinterpret_cast<int32_t *>(ws);
        p.ws_acc = reinterpret_cast<float *>(ws + size_t(grid) * 32);
        p.ws_ml = p.ws_acc + size_t(grid) * 2 * cols * HD;
    }
    launch_pdl(attend_paged_kernel<HD, NT>, grid, kThreadsC, geo<HD, NT>::total, s, p, map_k, map_v);
    if (cudaPeekAtLastError() != cudaSuccess) return FNB_LAUNCH_FAILED;
    if (fold) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(unsigned(grid - 1), unsigned(cols)), cfg.blockDim = dim3(kFoldWarps * 32), cfg.stream = s;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr, cfg.numAttrs = 1;
        (void) cudaLaunchKernelEx(&cfg, attend_paged_fold_kernel<HD, NT>, static_cast<const paged_params>(p));
    }
    return launch_status();
}
template <int HD>
int32_t launch_paged_hd(const fnb_attend_paged_args * a, paged_params & p, cudaStream_t s) {
    switch (column_blocks(a)) {
        case 1: return launch_paged<HD, 1>(a, p, s);
        case 2: return launch_paged<HD, 2>(a, p, s);
        case 4: return launch_paged<HD, 4>(a, p, s);
        default: return launch_paged<HD, 8>(a, p, s);
    }
}
template <int HD>
bool prepare_hd() { return configure<HD, 1>() && configure<HD, 2>() && configure<HD, 4>() && configure<HD, 8>(); }

}  // namespace

bool attend_paged_prepare_device() {
    (void) encode_tensor_map();
    return prepare_hd<256>() && prepare_hd<128>() && prepare_hd<64>();
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
    if (!one_tile(a) && (!ok_ptr(a->workspace, 16) || a->workspace_bytes < paged_workspace(a))) return FNB_REJECTED;
    paged_params p = {};
    p.q = a->q, p.gate = a->gate, p.k_scale = a->k_scale, p.v_scale = a->v_scale;
    p.table = a->table, p.n_cells = a->n_cells, p.row_start = a->row_start, p.out = a->out, p.err = a->err;
    p.cache_slots = a->cache_slots, p.rows = a->rows, p.n_req = a->n_req, p.max_pages = a->max_pages;
    const int64_t held = int64_t(a->max_pages) * a->page_size;
    p.cells_max = int(held < INT32_MAX - kTileCells ? held : INT32_MAX - kTileCells);
    p.n_pages = int(a->cache_slots / a->page_size), p.page_shift = __builtin_ctz(unsigned(a->page_size));
    p.n_q = a->n_q_heads, p.n_kv = a->n_kv_heads, p.group = a->n_q_heads / a->n_kv_heads;
    p.scale_log2 = a->scale * kLog2eF;
    p.e1024 = 0x64006400u, p.e64 = 0x54005400u;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->head_dim == 256) return launch_paged_hd<256>(a, p, s);
    return a->head_dim == 128 ? launch_paged_hd<128>(a, p, s) : launch_paged_hd<64>(a, p, s);
}
