// The KV4 cell format: a cache plane in 4 bits, groups of 32 values.
//   m     the group's value of largest magnitude (the positive one when m and -m both occur)
//   d     FP16(BF16(m / -8)), |d| <= 2720: an FP16 scale of at most eight significant bits
//   code  clamp(nearest-even(x id), -8, 7) + 8 with id = 1 / d in F32; all 8 when d is 0
//   value (code - 8) d
// Dividing by -8 gives the value of largest magnitude the code 0, so that all sixteen levels are in use (with a
// symmetric rule the sixteenth never is).  The scale keeps eight bits because a code less 8 has at most three more:
// their product is then EXACT in FP16, and attention can widen a cell to one FP16 operand instead of two (a rounded one
// and its residual, as it needs for the 8-bit formats).  Against a scale of eleven bits this moves a value by at most
// 2^-9 of itself, next to a quantisation step of 1/8 of the group's largest.  |d| stops at 2720 (values at 21760), so that
// a reader can widen in FP16 either way: subtract 8 first, as attention here does, or multiply first, as (code + 16) d - 24 d.
// A group that holds an infinity or a NaN gets the scale NaN: the fault shows in whatever reads the cell.
//
// Planes are head-major, [kv_head][slot][head_dim / 2] bytes and [kv_head][slot][head_dim / 32] FP16 scales: a page of
// one head is one contiguous run of either, which is what a bulk copy wants.  Codes lie two to a byte in the order of
// the values, low nibble first.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace fnb {

// the order in which a group's extreme is chosen: larger magnitude first, then the positive sign; as an unsigned number,
// so that a maximum over keys finds it, and so that infinities and NaN come out on top
__device__ __forceinline__ uint32_t kv4_key(float x) {
    const uint32_t u = __float_as_uint(x);
    return __funnelshift_l(u, u, 1) ^ 1u;
}
__device__ __forceinline__ uint32_t kv4_key4(float4 v) {
    return max(max(kv4_key(v.x), kv4_key(v.y)), max(kv4_key(v.z), kv4_key(v.w)));
}
template <int G>
__device__ __forceinline__ uint32_t group_max_key(uint32_t v) {
#pragma unroll
    for (int m = G / 2; m > 0; m >>= 1) v = max(v, __shfl_xor_sync(kFull, v, m));
    return v;
}

struct kv4_rule {
    uint16_t db;  // the scale's bits
    float id;
    __device__ __forceinline__ explicit kv4_rule(uint32_t key) {
        const float m = __uint_as_float((key >> 1) | (~key << 31));
        const float b = __bfloat162float(__float2bfloat16_rn(__fmul_rn(m, -0.125f)));
        const __half h = __float2half_rn(fminf(fmaxf(b, -2720.0f), 2720.0f));
        const float d = __half2float(h);
        const bool finite = key < 0xff000000u, some = d != 0.0f;
        db = !finite ? 0x7e00u : some ? __half_as_ushort(h) : 0u;
        id = finite && some ? __fdiv_rn(1.0f, d) : 0.0f;
    }
    // cvt.rni saturates and turns a NaN into 0
    __device__ __forceinline__ static uint32_t code(float x, float id) {
        return uint32_t(max(-8, min(7, __float2int_rn(__fmul_rn(x, id)))) + 8);
    }
    __device__ __forceinline__ static uint32_t code4(float4 v, float id) {  // four codes in sixteen bits
        return code(v.x, id) | (code(v.y, id) << 4) | (code(v.z, id) << 8) | (code(v.w, id) << 12);
    }
};

// four codes (the low sixteen bits of w) widened: a nibble under the exponent of 2^23 is 2^23 + code
__device__ __forceinline__ float4 kv4_widen4(uint32_t w, float d) {
    float4 r;
    r.x = __fmul_rn(__fadd_rn(__uint_as_float((w & 15u) | 0x4b000000u), -8388616.0f), d);
    r.y = __fmul_rn(__fadd_rn(__uint_as_float(((w >> 4) & 15u) | 0x4b000000u), -8388616.0f), d);
    r.z = __fmul_rn(__fadd_rn(__uint_as_float(((w >> 8) & 15u) | 0x4b000000u), -8388616.0f), d);
    r.w = __fmul_rn(__fadd_rn(__uint_as_float(((w >> 12) & 15u) | 0x4b000000u), -8388616.0f), d);
    return r;
}

}  // namespace fnb
