// Shared device helpers: exact scalar rules of the ggml block formats, warp reductions, memory-access hints.
// Every kernel in this library is HBM-bound; these helpers keep the arithmetic bit-exact with the CPU
// definition (separately rounded products and sums, IEEE division and square root) at no bandwidth cost.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/fnb200.h"

namespace fnb {

constexpr int kWarp = 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kSmCount = 148;  // B200: grids are sized in multiples of this

// ---- argument checks shared by the launchers ----------------------------------------------------------
inline bool aligned(const void * p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline bool ok_ptr(const void * p, size_t a) { return p != nullptr && aligned(p, a); }
inline bool ok_opt(const void * p, size_t a) { return p == nullptr || aligned(p, a); }

inline int32_t launch_status() {
    // cudaPeekAtLastError leaves the error in place for the caller, as the reference's launchers do
    return cudaPeekAtLastError() == cudaSuccess ? FNB_OK : FNB_LAUNCH_FAILED;
}

// ---- programmatic dependent launch ----------------------------------------------------------------------------------
// The kernels of the row-wise chain run back to back on one stream, each a few tens of microseconds at the shard sizes
// of a multi-GPU run, so the gap between two of them (grid launch, shared-memory carve-out, barrier set-up) shows.
// They are launched with programmatic stream serialisation: a kernel's CTAs may become resident while its predecessor
// drains; pdl_wait() returns once the predecessor has completed and its writes are visible, and MUST come before the
// kernel's first access to global memory (everything before it touches only registers, shared memory and launch
// arguments).  Every kernel launched this way executes pdl_wait(), which keeps completion transitive along the stream.
// pdl_launch_dependents() lets the successor's CTAs start as soon as every CTA of this grid has begun.  Without a
// programmatic predecessor or successor both are no-ops.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class... KArgs, class... Args>
inline void launch_pdl(void (*kernel)(KArgs...), int grid, int block, size_t smem, cudaStream_t s, Args &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(grid)), cfg.blockDim = dim3(unsigned(block));
    cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    (void) cudaLaunchKernelEx(&cfg, kernel, KArgs(args)...);  // the launcher reads the outcome with cudaPeekAtLastError
}

// number of CTAs for a grid-stride kernel: enough to fill the machine `waves` times, never more than the work
inline int grid_for(int64_t work_ctas, int ctas_per_sm) {
    const int64_t cap = int64_t(kSmCount) * ctas_per_sm;
    return int(work_ctas < cap ? (work_ctas > 0 ? work_ctas : 1) : cap);
}

// ---- global memory access with cache hints --------------------------------------------------------------
// Streaming data (read once, written once) bypasses L1 and is marked evict-first in L2 so the small reused
// state (weights, embedding table) keeps its L2 lines.
__device__ __forceinline__ float4 ld_stream(const float4 * p) { return __ldcs(p); }
__device__ __forceinline__ uint4 ld_stream(const uint4 * p) { return __ldcs(p); }
__device__ __forceinline__ void st_stream(float4 * p, float4 v) { __stcs(p, v); }
__device__ __forceinline__ void st_stream(uint4 * p, uint4 v) { __stcs(p, v); }
__device__ __forceinline__ void st_stream(uint2 * p, uint2 v) { __stcs(p, v); }
__device__ __forceinline__ void st_stream(uint32_t * p, uint32_t v) { __stcs(p, v); }

// ---- FP16 storage conversions ---------------------------------------------------------------------------
// F32 -> FP16 bits, round to nearest even, overflow to infinity; a NaN becomes sign | 0x7E00, which is what the
// CPU definition's conversion returns (cvt.rn.f16.f32 would give 0x7FFF).
__device__ __forceinline__ uint16_t f32_to_f16_bits(float f) {
    uint16_t h = __half_as_ushort(__float2half_rn(f));
    if (f != f) h = uint16_t(((__float_as_uint(f) >> 16) & 0x8000u) | 0x7e00u);
    return h;
}
__device__ __forceinline__ float f16_bits_to_f32(uint16_t h) { return __half2float(__ushort_as_half(h)); }

// ---- rounding rules ---------------------------------------------------------------------------------------
// (int8_t) roundf(v) for |v| < 2^23: roundf(v) = trunc(v + copysign(0.5 - 2^-25, v)) for every float in that
// range (checked exhaustively on the CPU), so the code is one logic op, one add and one convert.  NaN converts to 0,
// which is also the byte the CPU's convert leaves.  Only the low byte of the result is meaningful.
__device__ __forceinline__ int round_half_away_bits(float v) {
    const float h = __uint_as_float((__float_as_uint(v) & 0x80000000u) | 0x3effffffu);
    return __float2int_rz(__fadd_rn(v, h));
}

// ---- warp reductions ----------------------------------------------------------------------------------
__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
    int lo = __double2loint(v), hi = __double2hiint(v);
    lo = __shfl_xor_sync(kFull, lo, m);
    hi = __shfl_xor_sync(kFull, hi, m);
    return __hiloint2double(hi, lo);
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v = __dadd_rn(v, shfl_xor_f64(v, m));
    return v;
}
// max / sum over aligned groups of G lanes (G a power of two)
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int m = G / 2; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, m));
    return v;
}
template <int G>
__device__ __forceinline__ int group_sum(int v) {
#pragma unroll
    for (int m = G / 2; m > 0; m >>= 1) v += __shfl_xor_sync(kFull, v, m);
    return v;
}

// ---- the scalar rules of the 8-bit block formats ---------------------------------------------------------
// four int32 codes -> four packed int8 (low byte of each), and the sum of four packed int8
// ---- two FP32 operations per instruction (fma / mul / add .f32x2 of sm_100) ---------------------------------
// Each half of the pair is the IEEE round-to-nearest operation, so results are the scalar ones - unless a packed product goes
// into a packed sum and nowhere else: the compiler makes one FMA of the two, with one rounding, -fmad=false and the .rn of
// both notwithstanding (seen in every one of 65 536 pairs).  Where both roundings count, one of the two stays scalar, or the
// product has a second use, as in ggml_q8_rule::code4 (its codes are the scalar rule's over 4.5e9 values at the codes' borders).
// For kernels bound by instruction issue rather than by the FP32 pipe (SwiGLU: the written-out division is seven dependent
// FP32 operations per value) this halves those instructions.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpk(f32x2 v, float & x, float & y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// the low byte of each of four ints, whatever their range
__device__ __forceinline__ uint32_t pack4_low_bytes(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// For codes known to lie in [-128, 127] (or to be the 0 a NaN converts to): the saturating pack never saturates and
// takes two instructions a word where byte permutes take three (worth 4.5 % of the SwiGLU kernel's time).
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    uint32_t hi, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(hi) : "r"(d), "r"(c), "r"(0));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(b), "r"(a), "r"(hi));
    return w;
}
__device__ __forceinline__ int sum4_i8(uint32_t w) { return __dp4a(int(w), 0x01010101, 0); }

// ggml reference rule (Q8_0, Q8_1): d = amax / 127, id = d ? 1 / d : 0, q = (int8_t) roundf(x id).
// With a finite id the scaled value stays within +-127.5, where trunc(v + copysign(0.5 - 2^-25, v)) equals
// roundf(v) for every float (checked exhaustively), so the code is one add and one convert.  id is infinite only
// when d is a subnormal below 2^-128; then x id is +-inf or NaN, the CPU's convert gives INT32_MIN and the stored
// byte is 0 for every x - which id = 0 reproduces.
//
// The two divisions a block costs are written out for every amax in [2^-119, FLT_MAX]: d as the rounded product with
// rn(1 / 127) plus one exact-remainder correction, id as the hardware reciprocal estimate plus one Newton step.  Both
// are functions of one float, so "the same bits as the IEEE divisions" is checked by enumeration: every amax of that
// range, on the device, in the tests (d matches for every non-negative float; the reciprocal stops matching only below
// 2^-119, where d is subnormal and the estimate flushes it).  Zero, the tiny values, infinity and NaN take the
// divisions as written in the rule.
constexpr float kQ8RuleLow = 0x1p-119f, kQ8RuleHigh = 3.402823466e+38f;
struct ggml_q8_rule {
    float d, id;
    __device__ __forceinline__ explicit ggml_q8_rule(float amax) {
        if (amax >= kQ8RuleLow && amax <= kQ8RuleHigh) {
            constexpr float c = 1.0f / 127.0f;  // rn(1 / 127)
            const float q0 = __fmul_rn(amax, c);
            d = __fmaf_rn(__fmaf_rn(-127.0f, q0, amax), c, q0);
            float r0;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d));
            id = __fmaf_rn(r0, __fmaf_rn(-d, r0, 1.0f), r0);
        } else {
            d = __fdiv_rn(amax, 127.0f);
            const float r = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
            id = r < __uint_as_float(0x7f800000u) ? r : 0.0f;
        }
    }
    // only the low byte of the result is meaningful
    __device__ __forceinline__ int code(float x) const { return round_half_away_bits(__fmul_rn(x, id)); }
    // four codes packed into a word; the scaling and the rounding add run two values per instruction
    __device__ __forceinline__ uint32_t code4(float4 v) const {
        const f32x2 id2 = pk(id, id);
        float p[4], t[4];
        unpk(mul2(pk(v.x, v.y), id2), p[0], p[1]);
        unpk(mul2(pk(v.z, v.w), id2), p[2], p[3]);
        float h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __uint_as_float((__float_as_uint(p[i]) & 0x80000000u) | 0x3effffffu);
        unpk(add2(pk(p[0], p[1]), pk(h[0], h[1])), t[0], t[1]);
        unpk(add2(pk(p[2], p[3]), pk(h[2], h[3])), t[2], t[3]);
        return pack4(__float2int_rz(t[0]), __float2int_rz(t[1]), __float2int_rz(t[2]), __float2int_rz(t[3]));
    }
};
// the reference engine's activation rule: d = amax / 127, id = 127 / amax, q = nearest-even(x id) in +-127, NaN -> 0
// (cvt.rni.s32.f32 saturates an infinite product, which the clamp then takes to +-127, and turns NaN into 0)
struct act_rule {
    float d, id;
    __device__ __forceinline__ explicit act_rule(float amax) {
        d = __fdiv_rn(amax, 127.0f);
        id = amax > 0.0f ? __fdiv_rn(127.0f, amax) : 0.0f;
    }
    __device__ __forceinline__ int code(float x) const {
        return max(-127, min(127, __float2int_rn(__fmul_rn(x, id))));
    }
    __device__ __forceinline__ uint32_t code4(float4 v) const {
        const f32x2 id2 = pk(id, id);
        float p[4];
        unpk(mul2(pk(v.x, v.y), id2), p[0], p[1]);
        unpk(mul2(pk(v.z, v.w), id2), p[2], p[3]);
        return pack4(max(-127, min(127, __float2int_rn(p[0]))), max(-127, min(127, __float2int_rn(p[1]))),
                     max(-127, min(127, __float2int_rn(p[2]))), max(-127, min(127, __float2int_rn(p[3]))));
    }
};

// the reference engine's KV8 rule for one group of 64 values: scale = fp16_rn(amax / 127), s its F32 value,
// code = clamp(nearest-even(x / s), +-127) with an IEEE division, 0 when s is 0.  The division by the group's s is
// written out (reciprocal refined once per group, two exact-remainder corrections per value): the same quotient as
// __fdiv_rn for every FP16-representable s and |x| up to a few hundred s, without its per-call range check.
struct kv8_rule {
    uint16_t sb;
    float s, r;
    bool fast;
    __device__ __forceinline__ explicit kv8_rule(float amax) {
        sb = f32_to_f16_bits(__fdiv_rn(amax, 127.0f));
        s = f16_bits_to_f32(sb);
        fast = s >= 0x1p-24f && s <= 65504.0f;  // not 0, not infinite, not NaN
        float r0;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(fast ? s : 1.0f));
        r = __fmaf_rn(r0, __fmaf_rn(-s, r0, 1.0f), r0);
    }
    // cvt.rni saturates +-inf and maps NaN to 0; the clamp then gives the rule's +-127
    __device__ __forceinline__ int code_fast(float x) const {  // requires fast
        float q = __fmul_rn(x, r);
        q = __fmaf_rn(__fmaf_rn(-s, q, x), r, q);
        q = __fmaf_rn(__fmaf_rn(-s, q, x), r, q);
        return max(-127, min(127, __float2int_rn(q)));
    }
    __device__ __forceinline__ int code_any(float x) const {
        return s > 0.0f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x, s)))) : 0;
    }
    __device__ __forceinline__ int code(float x) const { return fast ? code_fast(x) : code_any(x); }
    // four values at once: one branch on the group's scale instead of one per value
    // (scalar on purpose: the two-values-per-instruction form made the rope kernel slower, 0.446 against 0.433 ms)
    __device__ __forceinline__ uint32_t code4(float4 v) const {
        if (fast) return pack4(code_fast(v.x), code_fast(v.y), code_fast(v.z), code_fast(v.w));
        return pack4(code_any(v.x), code_any(v.y), code_any(v.z), code_any(v.w));
    }
};

// Per-device, one-time kernel attribute set-up of the files that need more than 48 KB of shared memory; each
// returns false when the CUDA call fails.  fnb_prepare_device runs them all, so that no later launch has to.
bool glu_prepare_device();
bool rms_norm_quant_prepare_device();
bool rope_prepare_device();
bool expert_down_prepare_device();
bool expert_gate_up_prepare_device();
bool expert_down_iq4nl_prepare_device();
bool attend_prepare_device();
bool attend_paged_prepare_device();

}  // namespace fnb
