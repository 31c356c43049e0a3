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

// Where a head's blocks lie, one after the other at a step of `step` blocks, for a wave: everything here is
// the same in all lanes and little enough to stay in scalar registers.  Within a page (or a stream without
// pages) the pointers grow by additions; a page's place is worked out when its first block comes up, from an
// entry that was looked up when the page before began.
struct BlockWalk {
    typedef const __attribute__((address_space(4))) int32_t* table_ptr;
    const char *k, *v;
    const int8_t *ke, *ve;
    int32_t k_nb, v_nb, ke_nb, ve_nb;  // from block to block
    int32_t b, end;                    // the block; the first past the piece
    int32_t turn;                      // the first block of the next page (past the end without pages)
    int32_t entry;                     // its page

    __device__ __forceinline__ void place(const Kv8Tensor& tk, const Kv8Tensor& tv, int64_t unit, int i, int g) {
        k = tk.codes + unit * tk.nb[2] + (int64_t)i * tk.nb[0] + (int64_t)g * tk.nb[1];
        v = tv.codes + unit * tv.nb[2] + (int64_t)i * tv.nb[0] + (int64_t)g * tv.nb[1];
        ke = tk.exps + unit * tk.e_nb[2] + (int64_t)i * tk.e_nb[0] + (int64_t)g * tk.e_nb[1];
        ve = tv.exps + unit * tv.e_nb[2] + (int64_t)i * tv.e_nb[0] + (int64_t)g * tv.e_nb[1];
    }
    __device__ __forceinline__ int32_t look(const Kv8Pages& p, int s, int page) const {
        const int at = min(page, (end - 1) / kPageBlocks);
        return ((table_ptr)(uintptr_t)(p.pt + (int64_t)s * p.pt_stride))[at];
    }
    __device__ __forceinline__ void begin(const Kv8Pages& p, const Kv8Tensor& tk, const Kv8Tensor& tv, int s, int g, int first, int last) {
        b = first;
        end = last;
        k_nb = (int32_t)tk.nb[0];
        v_nb = (int32_t)tv.nb[0];
        ke_nb = (int32_t)tk.e_nb[0];
        ve_nb = (int32_t)tv.e_nb[0];
        turn = INT32_MAX;
        entry = 0;
        if (p.pt) {
            const int page = first / kPageBlocks;
            turn = (page + 1) * kPageBlocks;
            const int u = look(p, s, page);
            entry = look(p, s, page + 1);
            place(tk, tv, min(max(u, 0), p.n_pages - 1), first % kPageBlocks, g);
        } else {
            place(tk, tv, s, first, g);
        }
    }
    // On by `step` blocks (at most 8), where that is within the piece.
    __device__ __forceinline__ void go(const Kv8Pages& p, const Kv8Tensor& tk, const Kv8Tensor& tv, int s, int g, int step) {
        if (b + step >= end) return;
        b += step;
        if (b >= turn) {
            const int page = b / kPageBlocks;
            const int u = entry;
            entry = look(p, s, page + 1);
            place(tk, tv, min(max(u, 0), p.n_pages - 1), b % kPageBlocks, g);
            turn = (page + 1) * kPageBlocks;
        } else {
            k += (int64_t)step * k_nb;
            v += (int64_t)step * v_nb;
            ke += (int64_t)step * ke_nb;
            ve += (int64_t)step * ve_nb;
        }
    }
};

// Sum over the 64 lanes up to and including one's own (row shifts within 16 lanes, then the rows' last
// lanes broadcast); lane 63 holds the total.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr 1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
    return x;
}

// The larger of a value and its counterpart 32 lanes away (NaN if either is), and their sum, in both.
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

}  // namespace sixi
