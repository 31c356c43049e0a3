// kv8_device.hpp -- device helpers of the 8-bit cache's kernels.
#pragma once

#include "kv8_internal.hpp"

namespace sixi {

typedef float kv8_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t kv8_u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv8_f16x8 __attribute__((ext_vector_type(8)));

// 2^e for e in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) { return __builtin_bit_cast(float, (127 + e) << 23); }

__device__ __forceinline__ int clamp_exp(int e) { return min(max(e, SIXI_KV8_EXP_MIN), SIXI_KV8_EXP_MAX); }

// The smallest exponent in range with top <= 127 * 2^e: top = m * 2^k, 1 <= m < 2, fits 127 steps of
// 2^(k-6) up to m = 127/64.
__device__ __forceinline__ int scale_exp(float top) {
    const uint32_t u = __builtin_bit_cast(uint32_t, top);
    const int k = (int)(u >> 23) - 127;
    return clamp_exp(k - 6 + ((u & 0x7fffff) > 0x7e0000 ? 1 : 0));
}

// Byte offset of block b of stream s, and of its exponent (head 0).
__device__ __forceinline__ void block_at(const Kv8Pages& p, const int64_t (&nb)[3], const int64_t (&e_nb)[3], int s, int b,
                                         int64_t& at, int64_t& e_at) {
    if (p.pt) {
        const int page = min(max(p.pt[(int64_t)s * p.pt_stride + b / kPageBlocks], 0), p.n_pages - 1);
        at = (int64_t)page * nb[2] + (int64_t)(b % kPageBlocks) * nb[0];
        e_at = (int64_t)page * e_nb[2] + (int64_t)(b % kPageBlocks) * e_nb[0];
    } else {
        at = (int64_t)s * nb[2] + (int64_t)b * nb[0];
        e_at = (int64_t)s * e_nb[2] + (int64_t)b * e_nb[0];
    }
}

}  // namespace sixi
