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
//   K: ldmatrix hands a thread eight codes of a cell in one register.  A nibble at bits 0 .. 3 or 4 .. 7 of a half is the
//   FP16 SUBNORMAL code x 2^-24 or 16 code x 2^-24 as it stands, so one AND makes an operand register of two codes; the 16
//   is taken out of the queries (a power of two, exact).  The bias 8 sum(q) of a group enters as the accumulator's
//   initial value, the group's d multiplies its sum in F32: five logic instructions for eight codes.
//   V: ldmatrix.trans hands a thread four codes of each of two cells.  The bias cannot be taken out afterwards (over a
//   long flat row the sum of p (code - 8) is small against 8 sum(p)), so a nibble shifted to bits 6 .. 9 under the
//   exponent of 16 is 16 + code, and one fused multiply-add with d and -24 d gives (code - 8) d, exact in FP16 by the
//   format.  A warp owns one group of 32 dims, whose d it needs.
//   Queries and probabilities are split into two FP16 parts (the rounded value and its rounded residual), which keeps
//   what an F32 product would: errors against 64 bits are those of an F32 evaluation.  Queries are scaled by a power of
//   two per row so that their largest lies in [2^13, 2^14), probabilities by 2^14, which keeps both parts above FP16's
//   subnormals where it matters.  Softmax statistics are F32.
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
    static constexpr int kRing = (HD == 256 ? 5 : 8) * (NT <= 2 ? 1 : 2);
    static constexpr uint32_t kSwz = HD == 256 ? 7u : HD == 128 ? 3u : 1u;
    // shared memory
    static constexpr int ring = 0;
    static constexpr int prob = ring + kRing * kUnitBytes;      // uint4 [8 slabs][NT][32]
    static constexpr int bias = prob + 8 * NT * 512;            // float [kGroups][kCols]
    static constexpr int wmax = bias + kGroups * kCols * 4;     // float [8 warps][8]
    static constexpr int lsum = wmax + 256;                     // float [8 warps][8]
    static constexpr int corr = lsum + 256;                     // float [kCols]
    static constexpr int mfin = corr + kCols * 4;               // float [kCols]
    static constexpr int red = mfin + kCols * 4;                // float4: the other cell groups' accumulators
    static constexpr int bars = red + (kCellGroups - 1) * kGroups * 32 * kCols * 4;
    static constexpr int scan = bars + kRing * 8;               // int64 [16]: sums, then the start of this CTA's piece
    static constexpr int feed = scan + 16 * 8;                  // the feeder's walk
    static constexpr int total = feed + 64 + 1024;              // + slack to align the base to 1024 bytes
    static_assert(total * kCtas + 1024 * kCtas <= 233472, "shared memory of an SM");
};

struct paged_params {
    const float *q, *gate;
    const uint16_t *k_scale, *v_scale;
    const int32_t *table, *n_cells, *row_start;
    float * out;
    float *ws_acc, *ws_ml;
    int64_t * ws_head;  // [grid][4]: first unit of the piece, first unit and length of the item it starts in, packed item
    uint32_t * err;
    int64_t cache_slots;
    int64_t cells_max;  // what a table row can list
    int rows, n_req, max_pages, n_pages, page_shift, n_q, n_kv, group;
    float scale_log2;
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
__device__ __forceinline__ uint32_t h2_u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u32_h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }
// two F32 values as FP16 pairs: the rounded values and the rounded residuals
__device__ __forceinline__ void split2(float x, float y, uint32_t & hi, uint32_t & lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_u32(h);
    lo = h2_u32(__floats2half2_rn(__fsub_rn(x, f.x), __fsub_rn(y, f.y)));
}
// nibble moved to bits 6 .. 9 of each half -> (code - 8) d, with e = -24 d
__device__ __forceinline__ uint32_t widen2(uint32_t moved, __half2 d, __half2 e) {
    return h2_u32(__hfma2(u32_h2((moved & 0x03c003c0u) | 0x4c004c00u), d, e));
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
    int64_t units;
};
template <int COLS>
__device__ __forceinline__ request load_request(const paged_params & p, int r, bool report) {
    request x;
    int n = __ldg(p.n_cells + r);
    x.row0 = p.row_start != nullptr ? __ldg(p.row_start + r) : r;
    int end = p.row_start != nullptr ? __ldg(p.row_start + r + 1) : r + 1;
    if (report && p.err != nullptr && (n < 0 || int64_t(n) > p.cells_max || x.row0 < 0 || end < x.row0 || end > p.rows)) {
        atomicOr(p.err, FNB_ERR_PAGES);
    }
    n = n < 0 ? 0 : int64_t(n) > p.cells_max ? int(p.cells_max) : n;
    x.row0 = x.row0 < 0 ? 0 : x.row0;
    end = end > p.rows ? p.rows : end;
    x.n = n, x.m = end > x.row0 ? end - x.row0 : 0;
    x.tiles = n > 0 ? (n + kTileCells - 1) / kTileCells : 1;  // a request without cells still has rows to write
    x.blocks = int((int64_t(x.m) * p.group + COLS - 1) / COLS);
    x.units = int64_t(p.n_kv) * x.blocks * x.tiles;
    return x;
}

// the walk over a piece of the line: request, KV head, column block, tile
template <int COLS>
struct cursor {
    int r, h, blk, tile;
    request x;
    __device__ __forceinline__ void at(const paged_params & p, int request_index, int64_t offset) {
        r = request_index;
        x = load_request<COLS>(p, r, false);
        const int64_t per_head = int64_t(x.blocks) * x.tiles;
        h = int(offset / per_head);
        const int64_t rest = offset - h * per_head;
        blk = int(rest / x.tiles);
        tile = int(rest - int64_t(blk) * x.tiles);
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

// ---- the ring's feeder: warp 0's walk, kept in shared memory (its registers are the query fragments') ----------------
struct feeder {
    int r, h, blk, tile;
    int n, m, tiles, blocks;  // the walk's request
    int64_t issued, total;    // K and V tiles of the piece
    int stage;
};
// Issues the next tile of the piece, if there is one.  Warp 0, all lanes.  `slot` is this lane's page of the tile (set
// with the K tile, used again with the V tile), `id` its page id of the next one, fetched a tile ahead.
template <int HD, int NT>
__device__ __forceinline__ void feed_one(const paged_params & p, const CUtensorMap * map_k, const CUtensorMap * map_v, feeder * f,
                                         uint8_t * smem, uint64_t * full, int32_t & slot, int32_t & id, uint64_t policy) {
    using G = geo<HD, NT>;
    const int lane = threadIdx.x & 31;
    const int64_t k = f->issued;
    if (k >= f->total) return;
    const int page = 1 << p.page_shift, box = page < kTileCells ? page : kTileCells, boxes = kTileCells / box;
    const int base = f->tile * kTileCells, left = f->n - base, stage = f->stage, h = f->h;
    const int n_live = left <= 0 ? 0 : min(boxes, (left + box - 1) / box);
    const bool is_v = (k & 1) != 0;
    if (!is_v && lane < n_live) {
        if (id < 0 || id >= p.n_pages) {
            if (p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
            id = 0;
        }
        slot = int32_t((uint32_t(id) << p.page_shift) + uint32_t((base + lane * box) & (page - 1)));
    }
    uint8_t * st = smem + G::ring + stage * G::kUnitBytes;
    if (lane == 0) {
        mbar_expect_tx(&full[stage], uint32_t(n_live) * uint32_t(box) * (HD / 2 + G::kGroups * 2));
        mbar_arrive(&full[stage]);
    }
    __syncwarp();
    if (lane < n_live) {
        tensor_g2s(st + lane * box * (HD / 2), is_v ? map_v : map_k, slot, h, &full[stage], policy);
        const uint16_t * scale = (is_v ? p.v_scale : p.k_scale) + (int64_t(h) * p.cache_slots + slot) * G::kGroups;
        bulk_g2s(st + G::kCodeBytes + lane * box * G::kGroups * 2, scale, uint32_t(box) * G::kGroups * 2, &full[stage], policy);
    }
    if (is_v && k + 1 < f->total) {
        cursor<G::kCols> c;
        c.r = f->r, c.h = h, c.blk = f->blk, c.tile = f->tile;
        c.x.n = f->n, c.x.m = f->m, c.x.tiles = f->tiles, c.x.blocks = f->blocks;
        if (++c.tile >= c.x.tiles) c.next_item(p);
        __syncwarp();
        if (lane == 0) {
            f->r = c.r, f->h = c.h, f->blk = c.blk, f->tile = c.tile;
            f->n = c.x.n, f->m = c.x.m, f->tiles = c.x.tiles, f->blocks = c.x.blocks;
        }
        const int64_t cell = int64_t(c.tile) * kTileCells + lane * box;
        id = lane < boxes && cell < c.x.n ? __ldg(p.table + int64_t(c.r) * p.max_pages + (cell >> p.page_shift)) : -1;
    }
    __syncwarp();
    if (lane == 0) {
        f->issued = k + 1;
        f->stage = stage + 1 == G::kRing ? 0 : stage + 1;
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
    uint8_t * smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t * full = reinterpret_cast<uint64_t *>(smem + G::bars);
    feeder * s_feed = reinterpret_cast<feeder *>(smem + G::feed);
    int64_t * s_scan = reinterpret_cast<int64_t *>(smem + G::scan);   // [0 ..] warp sums, [10] units before the start
    volatile uint32_t * s_misc = reinterpret_cast<volatile uint32_t *>(s_scan + 12);  // [0] start request, [1] gave up
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
        if (r < p.n_req) mine += load_request<G::kCols>(p, r, blockIdx.x == 0).units;
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(kFull, upto, o);
        if (lane >= o) upto += up;
    }
    if (lane == 31) s_scan[wid] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < kWarpsC; ++w) {
        if (w < wid) upto += s_scan[w];
        total += s_scan[w];
    }
    const int64_t u0 = total * blockIdx.x / gridDim.x, u1 = total * (blockIdx.x + 1) / gridDim.x;
    if (u0 < u1 && upto > u0 && upto - mine <= u0) {  // one thread
        int64_t base = upto - mine;
        for (int j = 0; j < per; ++j) {
            const int64_t units = load_request<G::kCols>(p, tid * per + j, false).units;
            if (base + units > u0) {
                s_misc[0] = uint32_t(tid * per + j);
                s_scan[10] = base;
                break;
            }
            base += units;
        }
    }
    __syncthreads();
    if (tid == 0 && p.ws_head != nullptr) {
        int64_t * head = p.ws_head + int64_t(blockIdx.x) * 4;
        head[0] = u0;
        head[1] = total;
        if (u0 < u1) {
            cursor<G::kCols> c;
            c.at(p, int(s_misc[0]), u0 - s_scan[10]);
            head[2] = u0 - c.tile;                                                    // the item's first unit
            head[3] = (int64_t(c.x.tiles) << 32) | uint32_t(c.r);                     // its length, its request
            p.ws_ml[int64_t(gridDim.x) * 2 * G::kCols * 2 + blockIdx.x * 2] = __int_as_float(c.h);
            p.ws_ml[int64_t(gridDim.x) * 2 * G::kCols * 2 + blockIdx.x * 2 + 1] = __int_as_float(c.blk);
        }
    }
    if (u0 >= u1) return;

    cursor<G::kCols> c;
    c.at(p, int(s_misc[0]), u0 - s_scan[10]);

    // the ring is filled before anything else
    const uint64_t policy = l2_evict_first_policy();
    int32_t feed_slot = 0, feed_id = -1;  // warp 0's
    auto feed = [&]() {
        if (s_misc[1] == 0) feed_one<HD, NT>(p, &map_k, &map_v, s_feed, smem, full, feed_slot, feed_id, policy);
    };
    if (wid == 0) {
        const int page = 1 << p.page_shift, box = page < kTileCells ? page : kTileCells;
        const int64_t cell = int64_t(c.tile) * kTileCells + lane * box;
        feed_id = lane * box < kTileCells && cell < c.x.n ? __ldg(p.table + int64_t(c.r) * p.max_pages + (cell >> p.page_shift)) : -1;
        if (lane == 0) {
            s_feed->r = c.r, s_feed->h = c.h, s_feed->blk = c.blk, s_feed->tile = c.tile;
            s_feed->n = c.x.n, s_feed->m = c.x.m, s_feed->tiles = c.x.tiles, s_feed->blocks = c.x.blocks;
            s_feed->issued = 0, s_feed->total = 2 * (u1 - u0), s_feed->stage = 0;
        }
        __syncwarp();
        for (int k = 0; k < G::kRing; ++k) feed();
    }

    const int g = lane >> 2, t = lane & 3;
    const int nt = wid % NT, slab0 = wid / NT * NT;                  // scores: column block and first of NT slabs
    const int dg = wid % NB, cg = wid / NB;                          // outputs: dim group, cell group
    constexpr int kSlabs = 8 / G::kCellGroups;                       // slabs of a cell group
    float * s_bias = reinterpret_cast<float *>(smem + G::bias);
    float * s_wmax = reinterpret_cast<float *>(smem + G::wmax);
    float * s_lsum = reinterpret_cast<float *>(smem + G::lsum);
    float * s_corr = reinterpret_cast<float *>(smem + G::corr);
    float * s_mfin = reinterpret_cast<float *>(smem + G::mfin);
    uint4 * s_prob = reinterpret_cast<uint4 *>(smem + G::prob);
    // ldmatrix addresses inside a tile: this lane's row of the 16 cells, its chunk; the swizzle xors the chunk bits
    const int lrow = (lane & 7) + ((lane >> 3) & 1) * 8, lchunk = lane >> 4;

    int stage = 0;        // of the ring, and its phase's parity
    uint32_t parity = 0;
    int64_t u = u0;
    while (u < u1) {
        const int tile_first = c.tile;
        const int n_tiles = int(min(int64_t(c.x.tiles - c.tile), u1 - u));
        const bool whole = tile_first == 0 && n_tiles == c.x.tiles;
        const int col0 = c.blk * G::kCols;
        auto row_of_col = [&](int col) { return (col0 + col) / p.group; };

        // queries of column 8 nt + g: this lane's eight dims of every group, in the order of the fragments
        uint32_t qf[NB][8];  // per group: n0n1 hi b0 b1, lo b0 b1; n2n3 hi, lo
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
            const float up16 = __fmul_rn(up, 0.0625f);
            float sum[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                // dims 8 t + {0, 4}, {1, 5}, {2, 6}, {3, 7}: nibbles 0 .. 3 of the two halves of a cell's word; the odd
                // nibbles stand 16 times too high
                split2(__fmul_rn(v[b][0].x, up), __fmul_rn(v[b][1].x, up), qf[b][0], qf[b][2]);
                split2(__fmul_rn(v[b][0].y, up16), __fmul_rn(v[b][1].y, up16), qf[b][1], qf[b][3]);
                split2(__fmul_rn(v[b][0].z, up), __fmul_rn(v[b][1].z, up), qf[b][4], qf[b][6]);
                split2(__fmul_rn(v[b][0].w, up16), __fmul_rn(v[b][1].w, up16), qf[b][5], qf[b][7]);
                float s = 0.0f, s16 = 0.0f;  // what the fragments hold, summed
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 f = __half22float2(u32_h2(qf[b][j]));
                    if (j & 1) {
                        s16 += f.x + f.y;
                    } else {
                        s += f.x + f.y;
                    }
                }
                s = fmaf(s16, 16.0f, s);
                s += __shfl_xor_sync(kFull, s, 1);
                s += __shfl_xor_sync(kFull, s, 2);
                sum[b] = s;
            }
            if (slab0 == 0 && t == 0) {
#pragma unroll
                for (int b = 0; b < NB; ++b) s_bias[b * G::kCols + col] = sum[b] * -0x1p-21f;  // -8 x 2^-24
            }
            const float sc = fmaxf(p.scale_log2 * down * 0x1p24f, 0x1p-126f);
            sc0 = __shfl_sync(kFull, sc, 8 * t), sc1 = __shfl_sync(kFull, sc, 8 * t + 4);
            const int i0 = row_of_col(nt * 8 + 2 * t), i1 = row_of_col(nt * 8 + 2 * t + 1);
            lim0 = i0 < c.x.m ? c.x.n - c.x.m + i0 + 1 : 0, lim1 = i1 < c.x.m ? c.x.n - c.x.m + i1 + 1 : 0;
        }
        const int lim_min = c.x.n - c.x.m + row_of_col(0) + 1;   // cells every live row of the block sees
        named_barrier<1>(kThreadsC);                             // the bias is in place

        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        float acc[NT][2][4];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
#pragma unroll
                for (int z = 0; z < 4; ++z) acc[x][y][z] = 0.0f;
            }
        }

        for (int it = 0; it < n_tiles; ++it) {
            const int base = (tile_first + it) * kTileCells;
            const bool masked = base + kTileCells > lim_min;
            // ---- scores
            (void) ring_wait(&full[stage], parity, s_misc + 1, p.err);
            const uint8_t * kt = smem + G::ring + stage * G::kUnitBytes;
            if (++stage == G::kRing) stage = 0, parity ^= 1u;
            float sv[NT][4];
#pragma unroll
            for (int s = 0; s < NT; ++s) {
                const int row = (slab0 + s) * 16;
                uint16_t dk[2][NB];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint8_t * at = kt + G::kCodeBytes + (row + g + 8 * j) * (NB * 2);
                    if constexpr (NB == 8) {
                        *reinterpret_cast<uint4 *>(dk[j]) = *reinterpret_cast<const uint4 *>(at);
                    } else if constexpr (NB == 4) {
                        *reinterpret_cast<uint2 *>(dk[j]) = *reinterpret_cast<const uint2 *>(at);
                    } else {
                        *reinterpret_cast<uint32_t *>(dk[j]) = *reinterpret_cast<const uint32_t *>(at);
                    }
                }
                sv[s][0] = sv[s][1] = sv[s][2] = sv[s][3] = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    const uint32_t off = uint32_t(row + lrow) * (HD / 2) + uint32_t(b + lchunk) * 16;
                    uint32_t w[4];
                    ldm4(w, smem_u32(kt) + (off ^ (((off >> 7) & G::kSwz) << 4)));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float2 bi = *reinterpret_cast<const float2 *>(s_bias + (b + j) * G::kCols + nt * 8 + 2 * t);
                        float part[4] = {bi.x, bi.y, bi.x, bi.y};
                        uint32_t x0 = w[2 * j], x1 = w[2 * j + 1];
                        uint32_t a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
                        mma16816(part, a0, a1, a2, a3, qf[b + j][0], qf[b + j][1]);
                        mma16816(part, a0, a1, a2, a3, qf[b + j][2], qf[b + j][3]);
                        x0 >>= 8, x1 >>= 8;
                        a0 = x0 & 0x000f000fu, a1 = x1 & 0x000f000fu, a2 = x0 & 0x00f000f0u, a3 = x1 & 0x00f000f0u;
                        mma16816(part, a0, a1, a2, a3, qf[b + j][4], qf[b + j][5]);
                        mma16816(part, a0, a1, a2, a3, qf[b + j][6], qf[b + j][7]);
                        const float d0 = f16_bits_to_f32(dk[0][b + j]), d1 = f16_bits_to_f32(dk[1][b + j]);
                        sv[s][0] = fmaf(d0, part[0], sv[s][0]), sv[s][1] = fmaf(d0, part[1], sv[s][1]);
                        sv[s][2] = fmaf(d1, part[2], sv[s][2]), sv[s][3] = fmaf(d1, part[3], sv[s][3]);
                    }
                }
                if (masked) {
                    const int cell = base + row + g;
                    if (cell >= lim0) sv[s][0] = -INFINITY;
                    if (cell >= lim1) sv[s][1] = -INFINITY;
                    if (cell + 8 >= lim0) sv[s][2] = -INFINITY;
                    if (cell + 8 >= lim1) sv[s][3] = -INFINITY;
                }
            }
            // ---- maxima over the tile
            float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
            for (int s = 0; s < NT; ++s) t0 = fmaxf(t0, fmaxf(sv[s][0], sv[s][2])), t1 = fmaxf(t1, fmaxf(sv[s][1], sv[s][3]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) t0 = fmaxf(t0, __shfl_xor_sync(kFull, t0, o)), t1 = fmaxf(t1, __shfl_xor_sync(kFull, t1, o));
            if (g == 0) *reinterpret_cast<float2 *>(s_wmax + wid * 8 + 2 * t) = make_float2(t0, t1);
            named_barrier<1>(kThreadsC);  // also: nobody reads this tile's K stage or the last tile's V stage any more
            if (wid == 0) {
                if (it > 0 || u > u0) feed();
                feed();
            }
#pragma unroll
            for (int w = 0; w < 8 / NT; ++w) {
                const float2 v = *reinterpret_cast<const float2 *>(s_wmax + (w * NT + nt) * 8 + 2 * t);
                t0 = fmaxf(t0, v.x), t1 = fmaxf(t1, v.y);
            }
            const float n0 = fmaxf(m0, t0 * sc0), n1 = fmaxf(m1, t1 * sc1);
            const float f0 = n0 == -INFINITY ? 0.0f : n0, f1 = n1 == -INFINITY ? 0.0f : n1;
            float r0 = exp2f(m0 - f0), r1 = exp2f(m1 - f1);
            m0 = n0, m1 = n1;
            l0 *= r0, l1 *= r1;
            if (NT > 1 && slab0 == 0 && g == 0) *reinterpret_cast<float2 *>(s_corr + nt * 8 + 2 * t) = make_float2(r0, r1);
            // ---- probabilities into the second product's fragment order
#pragma unroll
            for (int s = 0; s < NT; ++s) {
                const float e0 = exp2f(fmaf(sv[s][0], sc0, kPShift - f0)), e1 = exp2f(fmaf(sv[s][1], sc1, kPShift - f1));
                const float e2 = exp2f(fmaf(sv[s][2], sc0, kPShift - f0)), e3 = exp2f(fmaf(sv[s][3], sc1, kPShift - f1));
                l0 += e0 + e2, l1 += e1 + e3;
                uint32_t h0, h1, q0, q1;
                split2(e0, e1, h0, q0);
                split2(e2, e3, h1, q1);
                s_prob[((slab0 + s) * NT + nt) * 32 + lane] =
                    make_uint4(transpose8x8(h0), transpose8x8(h1), transpose8x8(q0), transpose8x8(q1));
            }
            named_barrier<1>(kThreadsC);
            // ---- outputs
            (void) ring_wait(&full[stage], parity, s_misc + 1, p.err);
            const uint8_t * vt = smem + G::ring + stage * G::kUnitBytes;
            if (++stage == G::kRing) stage = 0, parity ^= 1u;
            const uint16_t * dv = reinterpret_cast<const uint16_t *>(vt + G::kCodeBytes) + dg;
#pragma unroll
            for (int x = 0; x < NT; ++x) {
                float2 f = make_float2(r0, r1);
                if (NT > 1) f = *reinterpret_cast<const float2 *>(s_corr + x * 8 + 2 * t);
#pragma unroll
                for (int y = 0; y < 2; ++y) acc[x][y][0] *= f.x, acc[x][y][1] *= f.y, acc[x][y][2] *= f.x, acc[x][y][3] *= f.y;
            }
            const int valid = min(kTileCells, c.x.n - base);    // cells of the tile that were copied
            bool fault = false;
#pragma unroll
            for (int sp = 0; sp < kSlabs; sp += 2) {
                const int sl = cg * kSlabs + sp;
                if (sl * 16 >= valid) break;
                // two slabs: matrices cells 0-7 and 8-15 of the first, then of the second
                const uint32_t off = uint32_t(sl * 16 + lrow + lchunk * 16) * (HD / 2) + uint32_t(dg) * 16;
                uint32_t w[4];
                ldm4t(w, smem_u32(vt) + (off ^ (((off >> 7) & G::kSwz) << 4)));
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int cell = (sl + j) * 16 + 2 * t;
                    uint16_t d[4] = {dv[cell * NB], dv[(cell + 1) * NB], dv[(cell + 8) * NB], dv[(cell + 9) * NB]};
                    if (masked) {
                        // behind the request's last cell lies whatever the memory held; a cell that holds no number
                        // is put back below for the rows that see it
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const bool in = cell + (z & 1) + (z >> 1) * 8 < valid, bad = (d[z] & 0x7c00u) == 0x7c00u;
                            fault = fault || (in && bad);
                            if (!in || bad) d[z] = 0;
                        }
                    }
                    const __half2 da = u32_h2(uint32_t(d[0]) | (uint32_t(d[1]) << 16)), db = u32_h2(uint32_t(d[2]) | (uint32_t(d[3]) << 16));
                    const __half2 k24 = __float2half2_rn(-24.0f);
                    const __half2 ea = __hmul2(da, k24), eb = __hmul2(db, k24);
                    const uint32_t x0 = w[2 * j], x1 = w[2 * j + 1];
                    const uint32_t a0 = widen2(x0 << 6, da, ea), a1 = widen2(x0 << 2, da, ea), a2 = widen2(x1 << 6, db, eb), a3 = widen2(x1 << 2, db, eb);
                    const uint32_t b0 = widen2(x0 >> 2, da, ea), b1 = widen2(x0 >> 6, da, ea), b2 = widen2(x1 >> 2, db, eb), b3 = widen2(x1 >> 6, db, eb);
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
                        const uint4 f = s_prob[((sl + j) * NT + x) * 32 + lane];
                        mma16816(acc[x][0], a0, a1, a2, a3, f.x, f.y);
                        mma16816(acc[x][1], b0, b1, b2, b3, f.x, f.y);
                        mma16816(acc[x][0], a0, a1, a2, a3, f.z, f.w);
                        mma16816(acc[x][1], b0, b1, b2, b3, f.z, f.w);
                    }
                }
            }
            if (masked && __any_sync(kFull, fault)) {
                for (int cell = cg * kSlabs * 16; cell < min(valid, (cg + 1) * kSlabs * 16); ++cell) {
                    if ((dv[cell * NB] & 0x7c00u) != 0x7c00u) continue;
#pragma unroll
                    for (int x = 0; x < NT; ++x) {
#pragma unroll
                        for (int z = 0; z < 2; ++z) {
                            if (base + cell >= c.x.n - c.x.m + row_of_col(x * 8 + 2 * t + z) + 1) continue;
#pragma unroll
                            for (int y = 0; y < 2; ++y) acc[x][y][z] = acc[x][y][z + 2] = NAN;
                        }
                    }
                }
            }
        }

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
        u += n_tiles;
        if (u < u1) c.next_item(p);
    }
    // after a wait that ran out: every copy has landed before the CTA's shared memory can be handed on
    if (tid == 0) {
        const int64_t k = s_feed->issued;
        for (int64_t j = 1; j <= G::kRing && j <= k; ++j) mbar_wait_landed(&full[(k - j) % G::kRing], uint32_t((k - j) / G::kRing) & 1u);
    }
}

// ---- the fold -----------------------------------------------------------------------------------------------------------
// Block (i, col): if the item that piece i + 1 starts inside of began in piece i, its pieces are folded for one column:
// weights 2^(m - max), accumulators and sums joined in the order of the pieces, eight warps taking every eighth piece.
constexpr int kFoldWarps = 8;
template <int HD, int NT>
__global__ void __launch_bounds__(kFoldWarps * 32) attend_paged_fold_kernel(const paged_params p, const int grid) {
    constexpr int COLS = 8 * NT, V = HD / 128 > 0 ? HD / 128 : 1;   // float4 vectors of a lane
    constexpr int LANES = HD / 4 < 32 ? HD / 4 : 32;
    __shared__ float4 s_acc[kFoldWarps][HD / 4];
    __shared__ float s_max[kFoldWarps], s_sum[kFoldWarps];
    pdl_launch_dependents();
    pdl_wait();
    const int i = blockIdx.x + 1, col = blockIdx.y;
    const int64_t * head = p.ws_head + int64_t(i) * 4;
    const int64_t u = __ldcg(head), total = __ldcg(head + 1);
    if (u >= total * (i + 1) / grid) return;                          // an empty piece
    const int64_t first = __ldcg(head + 2), packed = __ldcg(head + 3);
    if (first == u) return;                                           // piece i starts an item
    const int64_t len = packed >> 32;
    // The item began in piece b: the last one that does not start behind `first`.  Only the block of the first piece
    // behind b that is not empty folds.
    int64_t b = first * grid / total;
    while (total * (b + 1) / grid <= first) ++b;
    while (total * b / grid > first) --b;
    int64_t f = b + 1;
    while (f < i && total * (f + 1) / grid <= total * f / grid) ++f;
    if (f != i) return;
    const int r = int(uint32_t(packed));
    const int h = __float_as_int(__ldcg(p.ws_ml + int64_t(grid) * 2 * COLS * 2 + i * 2));
    const int blk = __float_as_int(__ldcg(p.ws_ml + int64_t(grid) * 2 * COLS * 2 + i * 2 + 1));
    const request x = load_request<COLS>(p, r, false);
    const int row = (blk * COLS + col) / p.group;
    if (row >= x.m) return;
    int64_t last = (first + len - 1) * grid / total;                  // the piece that holds the item's last unit
    while (total * (last + 1) / grid <= first + len - 1) ++last;
    while (total * last / grid > first + len - 1) --last;

    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    float4 acc[V];
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.0f;
    // the pieces after b hold the item from their start: slot 0; b's is its last: slot 1
#pragma unroll 4
    for (int64_t j = b + wid; j <= last; j += kFoldWarps) {
        if (total * (j + 1) / grid <= total * j / grid) continue;     // empty
        const int64_t slot = j * 2 + (j == b ? 1 : 0);
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(p.ws_ml + (slot * COLS + col) * 2));
        float4 a[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            a[v] = lane < LANES ? __ldcg(reinterpret_cast<const float4 *>(p.ws_acc + (slot * COLS + col) * HD) + lane + 32 * v)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.0f : top;
        const float wo = exp2f(m - base), wn = exp2f(ml.x - base);
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
        const float k = exp2f(s_max[w] - base);
        a = fmaf(reinterpret_cast<const float *>(s_acc[w])[d], k, a);
        s = fmaf(s_sum[w], k, s);
    }
    float y = s == 0.0f ? 0.0f : __fdiv_rn(a, s);
    const int64_t at = (int64_t(x.row0 + row) * p.n_q + h * p.group + (blk * COLS + col) % p.group) * HD + d;
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
    return grid * 2 * cols * (size_t(a->head_dim) + 2) * 4 + grid * 8 + grid * 32;
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
        p.ws_head = reinterpret_cast<int64_t *>(ws);
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
        (void) cudaLaunchKernelEx(&cfg, attend_paged_fold_kernel<HD, NT>, static_cast<const paged_params>(p), grid);
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
    p.cells_max = held < INT32_MAX - kTileCells ? held : INT32_MAX - kTileCells;
    p.n_pages = int(a->cache_slots / a->page_size), p.page_shift = __builtin_ctz(unsigned(a->page_size));
    p.n_q = a->n_q_heads, p.n_kv = a->n_kv_heads, p.group = a->n_q_heads / a->n_kv_heads;
    p.scale_log2 = a->scale * kLog2eF;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->head_dim == 256) return launch_paged_hd<256>(a, p, s);
    return a->head_dim == 128 ? launch_paged_hd<128>(a, p, s) : launch_paged_hd<64>(a, p, s);
}
