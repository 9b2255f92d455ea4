// Reading a KV4 plane back as F32 (kv4.cuh holds the format): out[t][h] = the head_dim values of slot cells[t] (or
// cell0 + t), kv head h.  Write-dominated like the 8-bit read-back: 144 bytes read and 1024 written per 256-value row.
// A warp takes kUnroll rows at a time; a lane takes four codes of a row (sixteen bits), so that every store instruction
// of the warp writes 512 contiguous bytes.  What it would wait for is a chain of two loads, the slot and the cell there,
// so the next rows' cells are under way while these are stored, and the slots of those after them.
#include "kv4.cuh"

namespace fnb {
namespace {

constexpr int kWarpsPerCta = 8;
constexpr int kUnroll = 2;
constexpr int kCtasPerSm = 5;  // 65 536 random slots of 2 x 256: 29.0 us (4: 29.4, 3: 32.5; four rows a warp: 33)

struct kv4_read_params {
    const uint8_t * codes;
    const uint16_t * scale;
    const int32_t * cells;  // [rows] or null: cell0 + row
    float * out;
    uint32_t * err;
    int64_t rows, cache_slots, cell0;
    int n_kv;
};

template <int HD>
__global__ void __launch_bounds__(kWarpsPerCta * 32) kv4_read_kernel(const kv4_read_params p) {
    pdl_wait();  // its start runs under the predecessor's end; its own successor starts when it ends (sooner: 31.5 us, not 29.0)
    constexpr int kUnits = HD / 4;                        // a row's runs of four codes
    constexpr int kLanes = kUnits < 32 ? kUnits : 32;     // lanes a row takes
    constexpr int kPer = kUnits / kLanes, kRows = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, rw = lane / kLanes;
    const int64_t warp = int64_t(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5);
    const int64_t step = int64_t(gridDim.x) * kWarpsPerCta * kUnroll * kRows;
    const int64_t n_rows = p.rows * p.n_kv;  // (row, head) pairs
    // slot and head of this lane's rows from `base` on; -1: none, or nothing to read there
    auto slots_of = [&](int64_t base, int64_t (&at)[kUnroll]) {
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int64_t r = base + j * kRows + rw;
            at[j] = -1;
            if (r >= n_rows) continue;
            const uint32_t t = uint32_t(r) / uint32_t(p.n_kv);   // rows x heads < 2^32
            const int h = int(uint32_t(r) - t * uint32_t(p.n_kv));
            const int64_t cell = p.cells != nullptr ? int64_t(__ldg(p.cells + t)) : p.cell0 + t;
            if (cell >= 0 && cell < p.cache_slots) {
                at[j] = int64_t(h) * p.cache_slots + cell;
            } else if (cell != -1 && sub == 0 && p.err != nullptr) {
                atomicOr(p.err, FNB_ERR_SLOT);
            }
        }
    };
    uint32_t w[kUnroll][kPer];
    uint16_t s[kUnroll][kPer];
    auto load = [&](const int64_t (&at)[kUnroll]) {
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (at[j] < 0) continue;
            const uint16_t * q = reinterpret_cast<const uint16_t *>(p.codes + at[j] * (HD / 2));
            const uint16_t * d = p.scale + at[j] * (HD / 32);
#pragma unroll
            for (int i = 0; i < kPer; ++i) w[j][i] = __ldg(q + sub + i * kLanes), s[j][i] = __ldg(d + (sub + i * kLanes) / 8);
        }
    };
    int64_t at[kUnroll], next[kUnroll];
    int64_t base = warp * kUnroll * kRows;
    if (base >= n_rows) return;
    slots_of(base, at);
    load(at);
    slots_of(base + step, next);
    while (true) {
        float4 v[kUnroll][kPer];
        bool live[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            live[j] = at[j] >= 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) v[j][i] = kv4_widen4(w[j][i], f16_bits_to_f32(s[j][i]));
        }
        const int64_t here = base;
        base += step;
        if (base < n_rows) {
#pragma unroll
            for (int j = 0; j < kUnroll; ++j) at[j] = next[j];
            load(at);
            slots_of(base + step, next);
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (!live[j]) continue;
            float4 * dst = reinterpret_cast<float4 *>(p.out + (here + j * kRows + rw) * HD);
#pragma unroll
            for (int i = 0; i < kPer; ++i) st_stream(dst + sub + i * kLanes, v[j][i]);
        }
        if (base >= n_rows) return;
    }
}

template <int HD>
void launch_read(const kv4_read_params & p, cudaStream_t s) {
    constexpr int64_t kPerWarp = int64_t(kUnroll) * (HD < 128 ? 128 / HD : 1);
    const int64_t warps = (p.rows * p.n_kv + kPerWarp - 1) / kPerWarp;
    launch_pdl(kv4_read_kernel<HD>, grid_for((warps + kWarpsPerCta - 1) / kWarpsPerCta, kCtasPerSm), kWarpsPerCta * 32, 0, s, p);
}

}  // namespace
}  // namespace fnb

extern "C" int32_t fnb_kv4_read_f32(const fnb_kv_read_args * a, void * stream) {
    using namespace fnb;
    if (a == nullptr || !ok_ptr(a->cache, 16) || !ok_ptr(a->scale, 16) || !ok_ptr(a->out, 16) || !ok_opt(a->cells, 4) ||
        !ok_opt(a->err, 4)) {
        return FNB_REJECTED;
    }
    if (a->rows < 1 || a->rows > INT32_MAX || a->cache_slots < 1 || a->cache_slots > INT32_MAX) return FNB_REJECTED;
    if (a->n_kv_heads < 1 || a->n_kv_heads > 256 || a->rows * a->n_kv_heads > int64_t(UINT32_MAX)) return FNB_REJECTED;
    if (a->cells == nullptr && (a->cell0 < 0 || a->cell0 > a->cache_slots - a->rows)) return FNB_REJECTED;
    kv4_read_params p;
    p.codes = static_cast<const uint8_t *>(a->cache), p.scale = a->scale, p.cells = a->cells, p.out = a->out, p.err = a->err;
    p.rows = a->rows, p.cache_slots = a->cache_slots, p.cell0 = a->cell0, p.n_kv = a->n_kv_heads;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a->head_dim) {
        case 256: launch_read<256>(p, s); break;
        case 128: launch_read<128>(p, s); break;
        case 64: launch_read<64>(p, s); break;
        default: return FNB_REJECTED;
    }
    return launch_status();
}
