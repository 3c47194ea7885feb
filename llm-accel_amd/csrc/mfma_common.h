// mfma_common.h -- byte planes and 16x16x64 products of the attention kernels
// that run on the matrix cores (internal to the library).
//
// K values enter clamped to [-2048, 2048] (attn_common.h) as k' = 256 a + b,
// b a signed byte; queries as q = 256 c + d + 128; probabilities p = 256 c + d
// with d a signed byte (c <= 64); V as K.  Operands of a product: lane l,
// byte b is row (position, head element or query) l % 16, contraction index
// 16 (l / 16) + b; its result: lane l, element s is row 4 (l / 16) + s of the
// first operand, row l % 16 of the second.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llm {
namespace {

typedef int32_t v4i __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int32_t med3(int32_t v, int32_t lo, int32_t hi) {
    return v < lo ? lo : (v > hi ? hi : v);
}
__device__ __forceinline__ uint32_t pack16(int32_t lo, int32_t hi) {
    return ((uint32_t)lo & 0xffffu) | ((uint32_t)hi << 16);
}
// Byte planes of four int16 values (two packed words): c = x >> 8 and
// d = (x & 255) - 128.
__device__ __forceinline__ uint32_t plane_c(uint32_t w0, uint32_t w1) {
    return __builtin_amdgcn_perm(w1, w0, 0x07050301u);
}
__device__ __forceinline__ uint32_t plane_d(uint32_t w0, uint32_t w1) {
    return __builtin_amdgcn_perm(w1, w0, 0x06040200u) ^ 0x80808080u;
}

__device__ __forceinline__ v4i mfma16(v4i a, v4i b, v4i c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
// 1 in each byte whose (a, b) bytes are those of 2048 = 256 * 8 + 0.
__device__ __forceinline__ v4i mask2048(v4i a, v4i b) {
    v4i r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t z = ((uint32_t)a[i] ^ 0x08080808u) | (uint32_t)b[i];
        const uint32_t nz = ((z & 0x7f7f7f7fu) + 0x7f7f7f7fu) | z;
        r[i] = (int32_t)((~nz >> 7) & 0x01010101u);
    }
    return r;
}
// Maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ int32_t quad_max(int32_t v) {
    const auto p = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = max((int32_t)p[0], (int32_t)p[1]);
    const auto q = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    return max((int32_t)q[0], (int32_t)q[1]);
}
__device__ __forceinline__ int32_t quad_sum(int32_t v) {
    const auto p = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = (int32_t)p[0] + (int32_t)p[1];
    const auto q = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    return (int32_t)q[0] + (int32_t)q[1];
}

}  // namespace
}  // namespace llm
