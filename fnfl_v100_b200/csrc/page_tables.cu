// Block tables, slot map and row positions of one step over a paged cache, built on the device from the requests'
// lengths, so that a step's host code needs no copy back and a captured graph serves every step.
//
// Request r holds n_old[r] cells in the pages its table row lists and gets n_new[r] more: its new pages come off the
// free list in the order of the requests, its rows follow those of the requests before it.  Both are exclusive sums
// over the requests.  What bounds it is latency: at 64 requests a few kilobytes move.  So ONE launch does all of it,
// and the sums over up to 2048 requests are formed by every CTA for itself (a few loads a thread), in preference to a
// second launch or to CTAs that wait on one another's sums.  The rows' and the new pages' requests are then found by
// bisection in shared memory, which costs the same whether one request has all the rows or every request one.
//
// n_cells may be n_old and free_head_out may be free_head, as a captured graph wants.  The CTAs of a launch therefore
// form one cluster and none writes before all have read (barrier.cluster); at most eight CTAs, so a few thousand rows a
// CTA in the largest steps, and one CTA (no cluster) up to kRowsOneCta rows.
#include "common.cuh"

namespace fnb {
namespace {

constexpr int kThreadsT = 1024;
constexpr int kMaxRequests = 2048;
constexpr int kPerThread = kMaxRequests / kThreadsT;
constexpr int kRowsOneCta = 1024;  // 4096 rows: one CTA 7.2 us, eight 5.2
constexpr int kClusterCtas = 8;

struct tables_params {
    const int32_t *n_old, *n_new, *free_pages, *free_head;
    int32_t *table, *n_cells, *row_start, *slots, *pos, *free_head_out;
    uint32_t * err;
    int64_t rows, n_free, cells_max;  // cells_max: what a table row can list
    int32_t n_req, max_pages, n_pages, page_shift;
};

// inclusive sum over the CTA's threads
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t * s_warp) {
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(kFull, v, o);
        if (lane >= o) v += up;
    }
    if (lane == 31) s_warp[wid] = v;
    __syncthreads();
    if (wid == 0) {
        int64_t w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(kFull, w, o);
            if (lane >= o) w += up;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    if (wid > 0) v += s_warp[wid - 1];
    __syncthreads();
    return v;
}

// the first request whose inclusive sum exceeds i (there is one)
__device__ __forceinline__ int owner_of(const int32_t * end, int n, int64_t i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (int64_t(end[mid]) > i) {
            hi = mid;
        } else {
            lo = mid + 1;
        }
    }
    return lo;
}

// ROWS: neighbouring rows a thread takes at a time, 1 or 4
template <int ROWS>
__global__ void __launch_bounds__(kThreadsT) page_tables_kernel(const tables_params p) {
    __shared__ int64_t s_warp[32];
    __shared__ int32_t s_row_end[kMaxRequests], s_page_end[kMaxRequests];
    __shared__ int32_t s_old[kMaxRequests];  // -1: the request gets nothing in this step
    __shared__ int32_t s_taken;
    pdl_launch_dependents();
    pdl_wait();

    const int tid = threadIdx.x, n_req = p.n_req;
    const int64_t page = int64_t(1) << p.page_shift;
    const int64_t head = p.free_head != nullptr ? int64_t(__ldcg(p.free_head)) : 0;
    const int64_t n_free = head >= 0 && head <= p.n_free ? p.n_free - head : 0;
    if (tid == 0) s_taken = 0;

    // a thread's requests: consecutive ones, so that the sums run in the requests' order
    int64_t old[kPerThread], fresh[kPerThread], grow[kPerThread];
    bool good[kPerThread];
    int64_t rows = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        old[j] = r < n_req ? int64_t(__ldcg(p.n_old + r)) : 0;
        fresh[j] = r < n_req ? int64_t(__ldcg(p.n_new + r)) : 0;
        good[j] = old[j] >= 0 && fresh[j] >= 0 && old[j] + fresh[j] <= p.cells_max;
        if (fresh[j] < 0) fresh[j] = 0;
        rows += fresh[j];
    }
    const int64_t rows_end = block_scan(rows, s_warp);
    int64_t row = rows_end - rows, pages = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        row += fresh[j];
        good[j] = good[j] && row <= p.rows;
        grow[j] = good[j] ? ((old[j] + fresh[j] + page - 1) >> p.page_shift) - ((old[j] + page - 1) >> p.page_shift) : 0;
        pages += grow[j];
        if (r < n_req) s_row_end[r] = int32_t(row < p.rows ? row : p.rows);
    }
    const int64_t pages_end = block_scan(pages, s_warp);
    int64_t at = pages_end - pages;
    bool fault = false;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        at += grow[j];
        if (r >= n_req) continue;
        good[j] = good[j] && (grow[j] == 0 || at <= n_free);
        s_page_end[r] = int32_t(at < INT32_MAX ? at : INT32_MAX);
        s_old[r] = good[j] ? int32_t(old[j]) : -1;
        if (good[j] && grow[j] > 0) atomicMax(&s_taken, int32_t(at));
        fault = fault || !good[j];
    }
    __syncthreads();
    if (gridDim.x > 1) {  // no CTA writes what another may still have to read
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }

    const int taken = s_taken;
    if (blockIdx.x == 0) {
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const int r = tid * kPerThread + j;
            if (r >= n_req) continue;
            p.n_cells[r] = int32_t(good[j] ? old[j] + fresh[j] : old[j]);
            p.row_start[r + 1] = s_row_end[r];
        }
        if (tid == 0) {
            p.row_start[0] = 0;
            if (p.free_head_out != nullptr) *p.free_head_out = int32_t(head + taken);
        }
        if (fault && p.err != nullptr) atomicOr(p.err, FNB_ERR_PAGES);
    }
    const int64_t first = int64_t(blockIdx.x) * kThreadsT + tid, step = int64_t(gridDim.x) * kThreadsT;
    // new pages into the table
    for (int64_t i = first; i < taken; i += step) {
        const int r = owner_of(s_page_end, n_req, i);
        const int64_t held = (int64_t(s_old[r]) + page - 1) >> p.page_shift;
        const int64_t j = i - (r > 0 ? int64_t(s_page_end[r - 1]) : 0);
        p.table[int64_t(r) * p.max_pages + held + j] = __ldg(p.free_pages + head + i);
    }
    // Rows; a page of this step is read off the free list, not from the table another thread is filling.  Neighbours mostly
    // share request and page, and so one search and one dependent load.
    const int64_t n_rows = s_row_end[n_req - 1];
    for (int64_t i0 = first * ROWS; i0 < p.rows; i0 += step * ROWS) {
        int32_t slot[ROWS], at_pos[ROWS];
        int r = -1;
        int64_t page_of = -1;   // the page that `id` belongs to
        int32_t id = -1;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int64_t i = i0 + k;
            slot[k] = -1, at_pos[k] = -1;
            if (i >= n_rows) continue;
            if (r < 0 || i >= s_row_end[r]) r = owner_of(s_row_end, n_req, i), page_of = -1;
            const int64_t o = s_old[r];
            if (o < 0) continue;
            const int64_t c = o + i - (r > 0 ? int64_t(s_row_end[r - 1]) : 0), j = c >> p.page_shift;
            if (j != page_of) {
                const int64_t held = (o + page - 1) >> p.page_shift;
                const int64_t share = r > 0 ? int64_t(s_page_end[r - 1]) : 0;
                id = j < held ? __ldcg(p.table + int64_t(r) * p.max_pages + j) : __ldg(p.free_pages + head + share + j - held);
                page_of = j;
            }
            at_pos[k] = int32_t(c);
            if (id >= 0 && id < p.n_pages) {
                slot[k] = int32_t((int64_t(id) << p.page_shift) + (c & (page - 1)));
            } else if (p.err != nullptr) {
                atomicOr(p.err, FNB_ERR_PAGES);
            }
        }
        auto put = [&](int32_t * to, const int32_t (&v)[ROWS]) {
            if constexpr (ROWS == 4) {
                if (i0 + 4 <= p.rows && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
                    *reinterpret_cast<int4 *>(to + i0) = make_int4(v[0], v[1], v[2], v[3]);
                    return;
                }
            }
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                if (i0 + k < p.rows) to[i0 + k] = v[k];
            }
        };
        put(p.slots, slot);
        put(p.pos, at_pos);
    }
}

}  // namespace
}  // namespace fnb

extern "C" int32_t fnb_page_tables(const fnb_page_tables_args * a, void * stream) {
    using namespace fnb;
    if (a == nullptr || !ok_ptr(a->n_old, 4) || !ok_ptr(a->n_new, 4) || !ok_ptr(a->table, 4) || !ok_ptr(a->n_cells, 4) ||
        !ok_ptr(a->row_start, 4) || !ok_ptr(a->slots, 4) || !ok_ptr(a->pos, 4) || !ok_opt(a->free_head, 4) ||
        !ok_opt(a->free_head_out, 4) || !ok_opt(a->err, 4)) {
        return FNB_REJECTED;
    }
    if (a->n_free < 0 || a->n_free > INT32_MAX || (a->n_free > 0 && !ok_ptr(a->free_pages, 4))) return FNB_REJECTED;
    if (a->n_req < 1 || a->n_req > kMaxRequests || a->max_pages < 1 || a->n_pages < 1) return FNB_REJECTED;
    if (a->rows < 1 || a->rows > INT32_MAX) return FNB_REJECTED;
    if (a->page_size < 1 || (a->page_size & (a->page_size - 1)) != 0) return FNB_REJECTED;
    if (int64_t(a->n_pages) * a->page_size > INT32_MAX) return FNB_REJECTED;
    tables_params p;
    p.n_old = a->n_old, p.n_new = a->n_new, p.free_pages = a->free_pages, p.free_head = a->free_head;
    p.table = a->table, p.n_cells = a->n_cells, p.row_start = a->row_start, p.slots = a->slots, p.pos = a->pos;
    p.free_head_out = a->free_head_out, p.err = a->err, p.rows = a->rows, p.n_free = a->n_free;
    p.n_req = a->n_req, p.max_pages = a->max_pages, p.n_pages = a->n_pages, p.page_shift = __builtin_ctz(unsigned(a->page_size));
    const int64_t held = int64_t(a->max_pages) * a->page_size;
    p.cells_max = held < INT32_MAX ? held : INT32_MAX;

    const int ctas = a->rows <= kRowsOneCta ? 1 : kClusterCtas;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas)), cfg.blockDim = dim3(kThreadsT), cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = unsigned(ctas), attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = ctas > 1 ? 2 : 1;
    // four rows at a time once each thread has several: 65 536 rows of 96 requests 10.0 us against 11.5
    (void) cudaLaunchKernelEx(&cfg, a->rows > int64_t(ctas) * kThreadsT ? page_tables_kernel<4> : page_tables_kernel<1>, p);
    return launch_status();
}
