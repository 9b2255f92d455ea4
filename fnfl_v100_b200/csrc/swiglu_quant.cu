// SwiGLU fused with requantisation of its output, and the stand-alone requantisers built from the same body.
//
//   v = (gate / (1 + expf(-gate))) * up            F32, expf bit-identical to the host C library's
//   every 32 values -> one block of the chosen 8-bit format
//
// HBM-bound by design: per 32 values 256 bytes are read (128 for a stand-alone requantiser) and 36 / 34 / 40
// written.  The tensors are dense and row-major with a block never crossing a row (cols is a multiple of 32),
// so the whole problem is one flat stream of blocks: block b reads values [32 b, 32 b + 32) and writes the b-th
// output block.  Rows do not appear in the kernel at all.
//
// The exact expf costs 12 FP64 operations as defined (8 as evaluated here) and the division 6 FP32 ones per value,
// so the kernel only stays memory-bound if everything around them costs almost nothing.  What ncu's instruction mix led to:
//
//   * ONE LANE OWNS ONE BLOCK.  amax, the code sum, d, 1/d and the FP16 header are computed once per 32 values
//     in-lane: no shuffles, no per-block work repeated by the lanes that share it (that repetition was ten
//     instructions per value when eight lanes shared a block).
//   * A lane's 128 bytes per operand are not a coalesced global access, so tiles are staged through shared memory
//     by cp.async.bulk: one producer lane streams tiles of 128 blocks (16 KiB per operand, each one contiguous run
//     in HBM) into a ring of five stages (six for the stand-alone requantisers, which stage one operand and keep
//     no table); sixteen consumer warps in four groups of four take the tiles in turn.  A lane reads its block's
//     eight 16-byte chunks in rotated order (chunk (j + lane) mod 8 at step j) so that the eight
//     lanes of a shared-memory phase hit 32 distinct banks; rotation is harmless because amax and the sum do not
//     care about order and each chunk's codes are written to that chunk's place.
//   * Finished blocks are assembled per warp in shared memory (36-byte stride: conflict-free) and leave as
//     aligned 128-bit stores.
//   * One range check per 128-bit vector selects a branch-free fast path (|gate| in [2^-40, 64): expf cannot hit
//     a special case, 1 + e < 2^93, the quotient is a normal number).  On it everything before the product with
//     `up` is a function of the gate alone, so a shortcut is admitted by enumerating every gate of the domain
//     against the generic path on the device: the division is reciprocal, one Newton step, product and ONE
//     exact-remainder correction (no range check, second correction or slow-path branch).  FP64 constants are
//     constant-bank operands, the 2^(i/32) table is in shared memory.
//
// Where that leaves it: about 35 warp instructions per 32 values, 8 of them FP64 (which occupy the dispatch port
// twice as long) and 4 on the conversion / special-function pipe.  The stand-alone requantisers (no expf) run at
// the HBM roofline; the GLU forms are bound by their arithmetic.
//
// All barrier waits are bounded; a wait that gives up sets FNB_ERR_TIMEOUT in the caller's error word (when one
// is given) and the CTA unwinds: consumers return, and the producer stays until every copy it issued has landed.
// One persistent CTA per SM.
#include <atomic>

#include "bulk_pipe.cuh"
#include "glu_math.cuh"

namespace fnb {
namespace {

enum class out_fmt { q8_1, q8_0, act };

#ifndef FNB_GLU_GROUPS
#define FNB_GLU_GROUPS 4
#endif
constexpr int kGroups = FNB_GLU_GROUPS;
#ifndef FNB_GLU_GROUP_WARPS
#define FNB_GLU_GROUP_WARPS 4
#endif
constexpr int kGroupWarps = FNB_GLU_GROUP_WARPS;
constexpr int kConsumerWarps = kGroups * kGroupWarps;
constexpr int kThreads = (kConsumerWarps + 1) * 32;
constexpr int kTileBlocks = kGroupWarps * 32;  // blocks per tile: 128 (16 KiB per operand)
#ifndef FNB_GLU_STAGES
#define FNB_GLU_STAGES 6
#endif
constexpr int kStages = FNB_GLU_STAGES;
#ifndef FNB_GLU_STAGES_GLU
#define FNB_GLU_STAGES_GLU 5
#endif
// the GLU forms stage two operands a tile and keep the 48 KiB exponential table: one stage fewer fits
__host__ __device__ constexpr int stages_of(bool glu) { return glu ? FNB_GLU_STAGES_GLU : kStages; }
static_assert(stages_of(false) >= kGroups && stages_of(true) >= kGroups,
              "a group's parity waits need a ring at least as deep as the number of groups");

template <out_fmt F>
struct fmt_traits;
template <>
struct fmt_traits<out_fmt::q8_1> {
    static constexpr int block_bytes = 36;
};
template <>
struct fmt_traits<out_fmt::q8_0> {
    static constexpr int block_bytes = 34;
};
template <>
struct fmt_traits<out_fmt::act> {
    static constexpr int block_bytes = 32;  // codes only; scales go to their own plane
};

__device__ __forceinline__ float amax4(float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); }

// F: output format; GLU: apply SwiGLU (else x = gate is quantised as is); F32OUT: also store v
template <out_fmt F, bool GLU, bool F32OUT>
__global__ void __launch_bounds__(kThreads, 1)
    glu_quant_kernel(const float * __restrict__ gate, const float * __restrict__ up, uint8_t * __restrict__ out,
                     float * __restrict__ scales, float * __restrict__ out_f32, int64_t n_blocks, uint32_t * err) {
    constexpr int BB = fmt_traits<F>::block_bytes;
    constexpr int kOperands = GLU ? 2 : 1;
    constexpr uint32_t kTileBytes = kTileBlocks * 128;  // per operand
    constexpr int kWarpOut = 32 * BB;                   // 1152 / 1088 / 1024 bytes: a multiple of 16
    constexpr int kStages = stages_of(GLU);
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_launch_dependents();
    uint8_t * data = smem;                                                     // [stages][operands][kTileBytes]
    uint8_t * outs = data + size_t(kStages) * kOperands * kTileBytes;          // [warps][kWarpOut]
    uint64_t * full = reinterpret_cast<uint64_t *>(outs + kConsumerWarps * kWarpOut);
    uint64_t * empty = full + kStages;
    unsigned long long * exp_tab = reinterpret_cast<unsigned long long *>(empty + kStages);  // GLU only

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kGroupWarps);
        }
        mbar_init_fence();
    }
    __syncthreads();  // nothing slow before this point: the producer starts streaming at once
    pdl_wait();       // the predecessor's writes are visible from here on; no global memory was touched before

    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    const int64_t n_tiles = (n_blocks + kTileBlocks - 1) / kTileBlocks;

    if (wid == kConsumerWarps) {
        // ---------------- producer: one lane streams the tiles ----------------
        if (lane != 0) return;
        hold_back_producer();
        const uint64_t policy = l2_evict_first_policy();
        int it = 0;
        bool ok = true;
        for (int64_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, ++it) {
            const int s = it % kStages;
            if (it >= kStages && !mbar_wait(&empty[s], (uint32_t(it / kStages) & 1u) ^ 1u, err)) {
                ok = false;
                break;
            }
            const int64_t b0 = tile * kTileBlocks;
            const uint32_t bytes = uint32_t(n_blocks - b0 < kTileBlocks ? n_blocks - b0 : kTileBlocks) * 128u;
            uint8_t * st = data + size_t(s) * kOperands * kTileBytes;
            mbar_expect_tx(&full[s], bytes * kOperands);
            bulk_g2s(st, gate + b0 * 32, bytes, &full[s], policy);
            if (GLU) bulk_g2s(st + kTileBytes, up + b0 * 32, bytes, &full[s], policy);
            mbar_arrive(&full[s]);
        }
        // The producer is the last to leave: every copy it issued must have landed before the CTA's shared memory
        // can be handed to another CTA.  When the consumers ran to the end these waits pass at once; after a wait
        // that gave up (here or in a consumer) they are what keeps the exit safe.
        (void) ok;
        for (int j = 1; j <= kStages && j <= it; ++j) {
            const int its = it - j;
            mbar_wait_landed(&full[its % kStages], uint32_t(its / kStages) & 1u);
        }
        return;
    }

    // ---------------- consumers: lane owns block `blk` of the tile ----------------
    if (GLU) {  // the exponential tables come out of constant memory while the first tiles are in flight
        load_exp2_table();
        glu_load_exp_table(exp_tab, threadIdx.x, kConsumerWarps * 32);
        named_barrier<1>(kConsumerWarps * 32);
    }
    const uint32_t tab_mid = smem_u32(exp_tab + kGluExpHalf);
    const int grp = wid / kGroupWarps, gw = wid - grp * kGroupWarps;
    const int blk = gw * 32 + lane;
    uint8_t * my_out = outs + wid * kWarpOut;

    int it = 0;
    for (int64_t tile = blockIdx.x; tile < n_tiles; tile += gridDim.x, ++it) {
        if (it % kGroups != grp) continue;
        const int s = it % kStages;
        const uint32_t fill = uint32_t(it / kStages);
        // A parity wait is only meaningful when the waiter is at most one phase ahead.  Successive fills of a stage
        // go to different groups here, so a fast group could reach its wait for fill n while fill n - 1 is still in
        // flight and read the stale "completed" parity of fill n - 2.  Waiting first for fill n - 1 to have been
        // CONSUMED (the empty barrier, which the producer's own ordering keeps within one phase) rules that out.
        if (fill > 0 && !mbar_wait(&empty[s], (fill - 1u) & 1u, err)) return;
        if (!mbar_wait(&full[s], fill & 1u, err)) return;
        const int64_t b0 = tile * kTileBlocks;
        const int64_t gb = b0 + blk;  // this lane's block in the tensor
        const bool live = gb < n_blocks;
        const uint8_t * st = data + size_t(s) * kOperands * kTileBytes + size_t(live ? blk : 0) * 128;

        float4 v[8];
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = (j + lane) & 7;  // rotated chunk: conflict-free across the lanes of a phase
            const float4 g = *reinterpret_cast<const float4 *>(st + 16 * c);
            if (GLU) {
                const float4 u = *reinterpret_cast<const float4 *>(st + kTileBytes + 16 * c);
                v[j] = glu4(g, u, tab_mid);  // a lane past the end works on block 0's data; nothing of it is stored
            } else {
                v[j] = g;
            }
            amax = fmaxf(amax, amax4(v[j]));
            if (F32OUT && live) st_stream(reinterpret_cast<float4 *>(out_f32 + gb * 32) + c, v[j]);
        }
        // the stage's bytes are in registers: hand it back before the arithmetic that remains
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);

        int qsum = 0;
        float d;
        if (F == out_fmt::q8_1) {
            const ggml_q8_rule rule(amax);
            uint32_t * o = reinterpret_cast<uint32_t *>(my_out) + 9 * lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = rule.code4(v[j]);
                qsum += sum4_i8(w);
                o[1 + ((j + lane) & 7)] = w;
            }
            d = rule.d;
            o[0] = uint32_t(f32_to_f16_bits(d)) | (uint32_t(f32_to_f16_bits(__fmul_rn(float(qsum), d))) << 16);
        } else if (F == out_fmt::q8_0) {
            const ggml_q8_rule rule(amax);
            uint16_t * o = reinterpret_cast<uint16_t *>(my_out) + 17 * lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = rule.code4(v[j]);
                const int c = (j + lane) & 7;
                o[1 + 2 * c] = uint16_t(w);
                o[2 + 2 * c] = uint16_t(w >> 16);
            }
            o[0] = f32_to_f16_bits(rule.d);
        } else {
            const act_rule rule(amax);
            uint32_t * o = reinterpret_cast<uint32_t *>(my_out) + 8 * lane;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t w = rule.code4(v[j]);
                qsum += sum4_i8(w);
                o[(j + lane) & 7] = w;
            }
            d = rule.d;
            if (live) {
                st_stream(reinterpret_cast<uint2 *>(scales) + gb,
                          make_uint2(__float_as_uint(d), __float_as_uint(__fmul_rn(d, float(qsum)))));
            }
        }
        __syncwarp();
        // the warp's 32 blocks leave as aligned 128-bit stores (a warp's output offset is a multiple of 16)
        const int64_t wb0 = b0 + gw * 32;
        const int64_t n_live = n_blocks - wb0;
        if (n_live >= 32) {
            uint4 * dst = reinterpret_cast<uint4 *>(out + wb0 * BB);
            for (int i = lane; i < kWarpOut / 16; i += 32) st_stream(dst + i, reinterpret_cast<const uint4 *>(my_out)[i]);
        } else if (n_live > 0) {  // ragged end of the tensor: 2-byte granules (every format's block size is even)
            uint8_t * dst = out + wb0 * BB;
            const int nbytes = int(n_live) * BB;
            for (int i = lane * 2; i < nbytes; i += 64) {
                *reinterpret_cast<uint16_t *>(dst + i) = *reinterpret_cast<const uint16_t *>(my_out + i);
            }
        }
        __syncwarp();
    }
}

template <out_fmt F, bool GLU>
constexpr size_t smem_bytes() {
    return size_t(stages_of(GLU)) * (GLU ? 2 : 1) * kTileBlocks * 128 + size_t(kConsumerWarps) * 32 * fmt_traits<F>::block_bytes +
           2 * stages_of(GLU) * 8 + (GLU ? kGluExpTableBytes : 0) + 64;
}

// raises the kernel's dynamic shared-memory limit once per device
template <out_fmt F, bool GLU, bool F32OUT>
bool ensure_configured() {
    static std::atomic<bool> configured[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    if (!configured[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(glu_quant_kernel<F, GLU, F32OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 int(smem_bytes<F, GLU>())) != cudaSuccess) {
            return false;
        }
        configured[dev].store(true, std::memory_order_release);
    }
    return true;
}

template <out_fmt F, bool GLU, bool F32OUT>
int32_t launch_one(const float * gate, const float * up, uint8_t * out, float * scales, float * out_f32, int64_t n_blocks,
                   uint32_t * err, cudaStream_t s) {
    constexpr size_t smem = smem_bytes<F, GLU>();
    if (!ensure_configured<F, GLU, F32OUT>()) return FNB_LAUNCH_FAILED;
    const int64_t n_tiles = (n_blocks + kTileBlocks - 1) / kTileBlocks;
    const int grid = int(n_tiles < kSmCount ? n_tiles : kSmCount);
    launch_pdl(glu_quant_kernel<F, GLU, F32OUT>, grid, kThreads, smem, s, gate, up, out, scales, out_f32, n_blocks, err);
    return launch_status();
}

template <out_fmt F, bool GLU>
int32_t launch(const float * gate, const float * up, void * out, float * scales, float * out_f32, int64_t rows,
               int32_t cols, uint32_t * err, cudaStream_t s) {
    if (!ok_ptr(gate, 16) || !ok_ptr(out, 16) || !ok_opt(out_f32, 16) || !ok_opt(err, 4)) return FNB_REJECTED;
    if (GLU && !ok_ptr(up, 16)) return FNB_REJECTED;
    if (F == out_fmt::act && !ok_ptr(scales, 8)) return FNB_REJECTED;
    if (rows < 1 || rows > INT32_MAX || cols < 32 || cols > (1 << 20) || cols % 32 != 0) return FNB_REJECTED;
    const int64_t n_blocks = rows * (cols / 32);
    uint8_t * o = static_cast<uint8_t *>(out);
    return out_f32 != nullptr ? launch_one<F, GLU, true>(gate, up, o, scales, out_f32, n_blocks, err, s)
                              : launch_one<F, GLU, false>(gate, up, o, scales, nullptr, n_blocks, err, s);
}

template <out_fmt F>
bool prepare_fmt() {
    return ensure_configured<F, true, false>() && ensure_configured<F, true, true>() && ensure_configured<F, false, false>() &&
           ensure_configured<F, false, true>();
}

}  // namespace

bool glu_prepare_device() {
    return prepare_fmt<out_fmt::q8_1>() && prepare_fmt<out_fmt::q8_0>() && prepare_fmt<out_fmt::act>();
}

}  // namespace fnb

using fnb::out_fmt;

extern "C" int32_t fnb_swiglu_q8_1(const float * gate, const float * up, void * out_q8_1, float * out_f32,
                                   int64_t rows, int32_t cols, uint32_t * err, void * stream) {
    return fnb::launch<out_fmt::q8_1, true>(gate, up, out_q8_1, nullptr, out_f32, rows, cols, err,
                                            static_cast<cudaStream_t>(stream));
}

extern "C" int32_t fnb_swiglu_act(const float * gate, const float * up, int8_t * codes, float * scales,
                                  float * out_f32, int64_t rows, int32_t cols, uint32_t * err, void * stream) {
    return fnb::launch<out_fmt::act, true>(gate, up, codes, scales, out_f32, rows, cols, err,
                                           static_cast<cudaStream_t>(stream));
}

extern "C" int32_t fnb_quantize_q8_1(const float * x, void * out_q8_1, int64_t rows, int32_t cols, uint32_t * err,
                                     void * stream) {
    return fnb::launch<out_fmt::q8_1, false>(x, nullptr, out_q8_1, nullptr, nullptr, rows, cols, err,
                                             static_cast<cudaStream_t>(stream));
}

extern "C" int32_t fnb_quantize_q8_0(const float * x, void * out_q8_0, int64_t rows, int32_t cols, uint32_t * err,
                                     void * stream) {
    return fnb::launch<out_fmt::q8_0, false>(x, nullptr, out_q8_0, nullptr, nullptr, rows, cols, err,
                                             static_cast<cudaStream_t>(stream));
}

extern "C" int32_t fnb_act_quantize(const float * x, int8_t * codes, float * scales, int64_t rows, int32_t cols,
                                    uint32_t * err, void * stream) {
    return fnb::launch<out_fmt::act, false>(x, nullptr, codes, scales, nullptr, rows, cols, err,
                                            static_cast<cudaStream_t>(stream));
}
