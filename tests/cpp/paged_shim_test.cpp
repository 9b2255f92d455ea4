// Host-side C++ test of the paged KV4 shims (include/fnb200_fn.hpp): three requests take two steps through page_tables,
// qsp_kv4 and attend_paged, state kept on the device; tables and slots are compared exactly, attention with a 64-bit
// evaluation over the cells that kv4_read returns.
//
//   paged_shim_test --reject     argument rejection only (runs without a GPU)
//   paged_shim_test              rejection + parity on the current CUDA device
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include <cuda_runtime.h>

#include "fnb200_fn.hpp"

static int g_fail = 0;
#define CHECK(cond)                                                              \
    do {                                                                         \
        if (!(cond)) {                                                           \
            std::fprintf(stderr, "FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_fail;                                                            \
        }                                                                        \
    } while (0)

template <typename T>
struct dev_buf {
    T * p = nullptr;
    size_t n;
    explicit dev_buf(size_t count, int fill = 0x5a) : n(count) {
        cudaMalloc(&p, n * sizeof(T));
        cudaMemset(p, fill, n * sizeof(T));
    }
    explicit dev_buf(const std::vector<T> & h) : dev_buf(h.size()) { up(h); }
    dev_buf(const dev_buf &) = delete;
    ~dev_buf() { cudaFree(p); }
    void up(const std::vector<T> & h) { cudaMemcpy(p, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice); }
    std::vector<T> down() const {
        std::vector<T> h(n);
        cudaMemcpy(h.data(), p, n * sizeof(T), cudaMemcpyDeviceToHost);
        return h;
    }
};

static void reject_cases() {
    float * a16 = reinterpret_cast<float *>(0x7f0000001000ull);  // aligned, never dereferenced
    uint16_t * s16 = reinterpret_cast<uint16_t *>(a16);
    int32_t * i16 = reinterpret_cast<int32_t *>(a16);
    fnb::qsa::qsp_kv_args k;
    k.kv_k = a16, k.kv_v = a16, k.pos = i16, k.rows = 4, k.max_cells = 64, k.k_cache = a16, k.v_cache = a16, k.theta_scale = 0.6f;
    k.k_scale = s16;  // one plane's scales alone
    CHECK(!fnb::qsa::qsp_kv4(k, nullptr));
    k.v_scale = s16, k.head_dim = 96;
    CHECK(!fnb::qsa::qsp_kv4(k, nullptr));
    CHECK(!fnb::qsa::kv4_read(a16, nullptr, nullptr, 0, 4, 64, 2, 256, a16, nullptr, nullptr));
    CHECK(!fnb::qsa::kv4_read(a16, s16, nullptr, 61, 4, 64, 2, 256, a16, nullptr, nullptr));
    fnb::qsa::page_tables_args t{};
    CHECK(!fnb::qsa::page_tables(t, nullptr));
    fnb::qsa::attend_paged_args a{};
    CHECK(fnb::qsa::attend_paged_workspace(a) == 0 && !fnb::qsa::attend_paged(a, nullptr));
}

static void parity_cases() {
    constexpr int R = 3, page = 16, n_pages = 12, slots = page * n_pages, max_pages = 20, n_q = 6, n_kv = 2, hd = 64, rows_max = 40;
    std::mt19937 rng(0x4b563470);
    std::normal_distribution<float> nd(0.0f, 1.0f);
    cudaStream_t s;
    cudaStreamCreate(&s);
    CHECK(fnb_prepare_device() == FNB_OK);
    dev_buf<int32_t> n_cells(std::vector<int32_t>{0, 0, 0}), n_new(R), head(std::vector<int32_t>{0}), free_pages(std::vector<int32_t>{7, 2, 11, 4, 0, 9});
    dev_buf<int32_t> table(size_t(R) * max_pages, 0xff), row_start(R + 1), slot(rows_max), pos(rows_max);
    dev_buf<uint8_t> kc(size_t(slots) * n_kv * hd / 2), vc(size_t(slots) * n_kv * hd / 2);
    dev_buf<uint16_t> ks(size_t(slots) * n_kv * hd / 32), vs(size_t(slots) * n_kv * hd / 32);
    dev_buf<uint32_t> err(std::vector<uint32_t>{0});

    const int steps[2][R] = {{20, 0, 5}, {1, 2, 12}};
    const std::vector<int32_t> want_cells[2] = {{20, 0, 5}, {21, 2, 17}};
    const std::vector<int32_t> want_start[2] = {{0, 20, 20, 25}, {0, 1, 3, 15}};
    const int want_head[2] = {3, 5};  // two pages and one; then one for the second request and one for the third's 17th cell
    for (int step = 0; step < 2; ++step) {
        n_new.up({steps[step][0], steps[step][1], steps[step][2]});
        fnb::qsa::page_tables_args t{};
        t.n_old = n_cells.p, t.n_new = n_new.p, t.free_pages = free_pages.p, t.free_head = head.p, t.table = table.p, t.n_cells = n_cells.p;
        t.row_start = row_start.p, t.slots = slot.p, t.pos = pos.p, t.free_head_out = head.p, t.err = err.p;
        t.rows = rows_max, t.n_free = 6, t.n_req = R, t.max_pages = max_pages, t.n_pages = n_pages, t.page_size = page;
        CHECK(fnb::qsa::page_tables(t, s));

        std::vector<float> q(size_t(rows_max) * n_q * hd), k(size_t(rows_max) * n_kv * hd), v(k.size());
        for (auto & x : q) x = nd(rng);
        for (auto & x : k) x = nd(rng);
        for (auto & x : v) x = nd(rng);
        dev_buf<float> dq(q), dk(k), dv(v), q_out(q.size()), out(q.size());
        fnb::qsa::qsp_kv_args a;
        a.q = dq.p, a.kv_k = dk.p, a.kv_v = dv.p, a.pos = pos.p, a.cells = slot.p, a.rows = rows_max, a.max_cells = slots;
        a.n_q_heads = n_q, a.n_kv_heads = n_kv, a.head_dim = hd, a.n_rot = 32, a.theta_scale = fnb_rope_theta_scale(1e6f, 32);
        a.q_out = q_out.p, a.k_cache = kc.p, a.v_cache = vc.p, a.k_scale = ks.p, a.v_scale = vs.p, a.err = err.p;
        CHECK(fnb::qsa::qsp_kv4(a, s));

        fnb::qsa::attend_paged_args at{};
        at.q = q_out.p, at.k_cache = kc.p, at.v_cache = vc.p, at.k_scale = ks.p, at.v_scale = vs.p, at.table = table.p;
        at.n_cells = n_cells.p, at.row_start = row_start.p, at.out = out.p, at.err = err.p, at.cache_slots = slots, at.rows = rows_max;
        at.n_req = R, at.max_pages = max_pages, at.page_size = page, at.max_rows = 20, at.n_q_heads = n_q, at.n_kv_heads = n_kv;
        at.head_dim = hd, at.scale = 0.125f;
        const size_t ws = fnb::qsa::attend_paged_workspace(at);
        dev_buf<uint8_t> work(ws);
        at.workspace = work.p, at.workspace_bytes = ws;
        CHECK(fnb::qsa::attend_paged(at, s));
        cudaStreamSynchronize(s);

        const std::vector<int32_t> cells = n_cells.down(), start = row_start.down(), tab = table.down(), sl = slot.down(), ps = pos.down();
        CHECK(cells == want_cells[step]);
        CHECK(start == want_start[step]);
        CHECK(head.down()[0] == want_head[step]);
        CHECK(err.down()[0] == 0);
        for (int r = 0; r < R; ++r) {
            for (int i = start[r]; i < start[r + 1]; ++i) {
                const int c = cells[r] - (start[r + 1] - start[r]) + (i - start[r]);
                CHECK(ps[i] == c && sl[i] == tab[r * max_pages + c / page] * page + c % page);
            }
        }
        CHECK(sl[start[R]] == -1 && sl[rows_max - 1] == -1 && ps[rows_max - 1] == -1);

        // the cells, in the order of the slots, and 64-bit attention over them
        dev_buf<float> kf(size_t(slots) * n_kv * hd), vf(kf.n);
        CHECK(fnb::qsa::kv4_read(kc.p, ks.p, nullptr, 0, slots, slots, n_kv, hd, kf.p, err.p, s));
        CHECK(fnb::qsa::kv4_read(vc.p, vs.p, nullptr, 0, slots, slots, n_kv, hd, vf.p, err.p, s));
        cudaStreamSynchronize(s);
        const std::vector<float> hk = kf.down(), hv = vf.down(), hq = q_out.down(), got = out.down();
        for (int r = 0; r < R; ++r) {
            for (int i = start[r]; i < start[r + 1]; ++i) {
                const int seen = ps[i] + 1;
                for (int h = 0; h < n_q; ++h) {
                    const float * qr = &hq[(size_t(i) * n_q + h) * hd];
                    std::vector<double> p(seen);
                    double top = -INFINITY, sum = 0, size = 0, big = 0;
                    auto at_cell = [&](int c) { return (size_t(tab[r * max_pages + c / page] * page + c % page) * n_kv + h / (n_q / n_kv)) * hd; };
                    for (int c = 0; c < seen; ++c) {
                        double dot = 0, mag = 0;
                        for (int d = 0; d < hd; ++d) {
                            const double x = double(qr[d]) * hk[at_cell(c) + d];
                            dot += x, mag += std::fabs(x);
                            big = std::fmax(big, std::fabs(double(hv[at_cell(c) + d])));
                        }
                        p[c] = dot * at.scale, top = std::fmax(top, p[c]), size = std::fmax(size, mag * at.scale);
                    }
                    for (auto & x : p) x = std::exp(x - top), sum += x;
                    // A score is a sum of hd products, each off by 2^-22 of itself at most (the split) and 2^-24 of the
                    // running sum per addition; its error moves a weight by the factor e^error, numerator and denominator
                    // alike.  A weight's exponential, its split and the output's sum of `seen` add 2^-20 for these lengths.
                    const double tol = 2 * big * (std::expm1(size * (hd + 4) * 0x1p-24) + 0x1p-20);
                    double worst = 0;
                    for (int d = 0; d < hd; ++d) {
                        double o = 0;
                        for (int c = 0; c < seen; ++c) o += p[c] * hv[at_cell(c) + d];
                        worst = std::fmax(worst, std::fabs(o / sum - got[(size_t(i) * n_q + h) * hd + d]));
                    }
                    CHECK(worst <= tol);
                }
            }
        }
        uint32_t bits;  // rows behind the last request's are left as they were
        std::memcpy(&bits, &got[size_t(start[R]) * n_q * hd], 4);
        CHECK(bits == 0x5a5a5a5au);
    }
    cudaStreamDestroy(s);
}

int main(int argc, char ** argv) {
    reject_cases();
    if (!(argc > 1 && std::strcmp(argv[1], "--reject") == 0)) {
        int n = 0;
        if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
            std::fprintf(stderr, "paged_shim_test: no CUDA device\n");
            return 2;
        }
        parity_cases();
    }
    std::printf("paged_shim_test: %s\n", g_fail == 0 ? "ok" : "FAILED");
    return g_fail == 0 ? 0 : 1;
}
