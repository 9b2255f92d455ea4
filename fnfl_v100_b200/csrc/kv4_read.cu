// Reading a KV4 plane back as F32 (kv4.cuh holds the format): out[t][h] = the head_dim values of slot cells[t] (or
// cell0 + t), kv head h.  Write-dominated like the 8-bit read-back: 144 bytes read and 1024 written per 256-value row.
// A warp takes a row; a lane takes four codes at a time (sixteen bits), so that every store instruction of the warp
// writes 512 contiguous bytes, and has kUnroll rows' loads in flight before it widens the first.
#include "kv4.cuh"

namespace fnb {
namespace {

constexpr int kWarpsPerCta = 8;
constexpr int kUnroll = 4;

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
    constexpr int kUnits = HD / 4;                        // a row's runs of four codes
    constexpr int kLanes = kUnits < 32 ? kUnits : 32;     // lanes a row takes
    constexpr int kPer = kUnits / kLanes, kRows = 32 / kLanes;
    const int lane = threadIdx.x & 31, sub = lane % kLanes, rw = lane / kLanes;
    const int64_t warp = int64_t(blockIdx.x) * kWarpsPerCta + (threadIdx.x >> 5);
    const int64_t n_warps = int64_t(gridDim.x) * kWarpsPerCta;
    const int64_t n_rows = p.rows * p.n_kv;  // (row, head) pairs
    for (int64_t base = warp * kUnroll * kRows; base < n_rows; base += n_warps * kUnroll * kRows) {
        uint32_t w[kUnroll][kPer];
        float s[kUnroll][kPer];
        bool live[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            const int64_t r = base + j * kRows + rw;
            live[j] = false;
            if (r >= n_rows) continue;
            const int64_t t = r / p.n_kv;
            const int h = int(r - t * p.n_kv);
            const int64_t cell = p.cells != nullptr ? int64_t(__ldg(p.cells + t)) : p.cell0 + t;
            if (cell < 0 || cell >= p.cache_slots) {
                if (cell != -1 && sub == 0 && p.err != nullptr) atomicOr(p.err, FNB_ERR_SLOT);
                continue;
            }
            live[j] = true;
            const int64_t c = int64_t(h) * p.cache_slots + cell;
            const uint16_t * q = reinterpret_cast<const uint16_t *>(p.codes + c * (HD / 2));
            const uint16_t * d = p.scale + c * (HD / 32);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                w[j][i] = __ldg(q + sub + i * kLanes);
                s[j][i] = f16_bits_to_f32(__ldg(d + (sub + i * kLanes) / 8));
            }
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
            if (!live[j]) continue;
            float4 * dst = reinterpret_cast<float4 *>(p.out + (base + j * kRows + rw) * HD);
#pragma unroll
            for (int i = 0; i < kPer; ++i) st_stream(dst + sub + i * kLanes, kv4_widen4(w[j][i], s[j][i]));
        }
    }
}

template <int HD>
void launch_read(const kv4_read_params & p, cudaStream_t s) {
    constexpr int64_t kPerWarp = int64_t(kUnroll) * (HD < 128 ? 128 / HD : 1);
    const int64_t warps = (p.rows * p.n_kv + kPerWarp - 1) / kPerWarp;
    kv4_read_kernel<HD><<<grid_for((warps + kWarpsPerCta - 1) / kWarpsPerCta, 32), kWarpsPerCta * 32, 0, s>>>(p);
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
    if (a->n_kv_heads < 1 || a->n_kv_heads > 256) return FNB_REJECTED;
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
