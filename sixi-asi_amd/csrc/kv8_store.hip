// kv8_store.hip -- rows into the 8-bit cache and back (include/sixi_kv8.h).
//
// One work-group per (stream, head, K or V, block of 32 cells).  A block's scale is a power of two:
//   e = min { e : max |x| <= 127 * 2^e },  code = rne(x * 2^-e),
// so multiplying by 2^-e is exact and the code is the value's nearest multiple whoever forms it.  A
// block that keeps cells in front of the new rows takes e' = max(e, its own) and shifts the kept codes
// by e' - e with one more rounding; its own exponent never falls until the block is begun anew.
//
// Bound by HBM: rows in once, codes out once; a block that is only partly written is read first (4 or
// 8 KiB), which is what a step that appends one token costs.  The new codes go through LDS in the
// cache's own order (K [D/16][32][16], V [D][32]), so that every store to the cache is 16 bytes and a
// whole block leaves as one piece.
#include "kv8_device.hpp"

namespace sixi {
namespace {

constexpr int kThreads = 256;

// 8 consecutive elements of a row as f32
__device__ __forceinline__ void load8(const char* p, bool f16, float (&x)[8]) {
    if (f16) {
        const kv8_f16x8 h = *reinterpret_cast<const kv8_f16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
    } else {
        const kv8_f32x4 a = *reinterpret_cast<const kv8_f32x4*>(p), b = *reinterpret_cast<const kv8_f32x4*>(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    }
}

__device__ __forceinline__ int code_of(float x, float inv) {
    // NaN fails both comparisons of the clamp's operands: stored as 0
    const float y = rintf(x * inv);
    return x == x ? (int)fminf(fmaxf(y, -127.0f), 127.0f) : 0;
}

// The rows of stream s that have a cell: cells [lo, hi), row 0 at cell `first`.
struct Span {
    int64_t first, lo, hi;
};
__device__ __forceinline__ Span span_of(const Kv8RowsArgs& a, int s) {
    Span r;
    r.first = a.kv_len ? a.kv_len[s] : 0;
    const int n = a.q_len ? min(max(a.q_len[s], 0), a.n_rows) : a.n_rows;
    const int64_t cells = (int64_t)a.pages.n_blocks * kBlk;
    r.lo = r.first > 0 ? r.first : 0;
    r.hi = r.first + n < cells ? r.first + n : cells;
    return r;
}

template <int D>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(Kv8RowsArgs a) {
    constexpr int kChunks = kBlk * D / 8 / kThreads;   // 8-element pieces of rows per thread
    constexpr int kVecs = kBlk * D / 16 / kThreads;    // 16-byte pieces of codes per thread
    __shared__ __align__(16) uint8_t codes[kBlk * D];
    __shared__ float tops[kThreads / 64];
    const int tid = threadIdx.x, s = blockIdx.z, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const Span r = span_of(a, s);
    const int64_t b64 = r.lo / kBlk + blockIdx.x;
    if (r.lo >= r.hi || b64 * kBlk >= r.hi) return;
    const int b = (int)b64;
    const int64_t cell0 = b64 * kBlk;
    const int c0 = r.lo > cell0 ? (int)(r.lo - cell0) : 0;
    const int c1 = r.hi < cell0 + kBlk ? (int)(r.hi - cell0) : kBlk;
    const Kv8Tensor& t = a.t[which];
    int64_t at, e_at;
    block_at(a.pages, t.nb, t.e_nb, s, b, at, e_at);
    char* block = t.codes + at + (int64_t)head * t.nb[1];
    int8_t* exp_p = t.exps + e_at + (int64_t)head * t.e_nb[1];

    kv8_u32x4 old[kVecs];
    const bool whole = c0 == 0 && c1 == kBlk;
    if (!whole) {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) old[i] = *reinterpret_cast<const kv8_u32x4*>(block + (tid + i * kThreads) * 16);
    }
    const int was = c0 > 0 ? clamp_exp(*exp_p) : SIXI_KV8_EXP_MIN;

    const char* rows = a.rows[which] + (int64_t)head * a.r_nb2[which] + (int64_t)s * a.r_nb3[which];
    float x[kChunks][8];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int id = tid + i * kThreads, c = id / (D / 8), d8 = id % (D / 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
        if (c >= c0 && c < c1) {
            const int64_t row = cell0 + c - r.first;
            load8(rows + row * a.r_nb1[which] + (int64_t)d8 * (a.f16[which] ? 16 : 32), a.f16[which] != 0, x[i]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = fabsf(x[i][e]);
            top = fmaxf(top, m < __builtin_huge_valf() ? m : 0.0f);  // finite values only (NaN compares false)
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    if (tid % 64 == 0) tops[tid / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const int e = max(scale_exp(top), was);
    const float inv = exp2_int(-e);

#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int id = tid + i * kThreads, c = id / (D / 8), d = id % (D / 8) * 8;
        if (c < c0 || c >= c1) continue;
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lo |= (uint32_t)(code_of(x[i][k], inv) & 0xff) << (8 * k);
            hi |= (uint32_t)(code_of(x[i][4 + k], inv) & 0xff) << (8 * k);
        }
        if (which == 0) {
            *reinterpret_cast<kv8_u32x2*>(codes + d / 16 * (kBlk * 16) + c * 16 + d % 16) = kv8_u32x2{lo, hi};
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                codes[(d + k) * kBlk + c] = (uint8_t)(lo >> (8 * k));
                codes[(d + 4 + k) * kBlk + c] = (uint8_t)(hi >> (8 * k));
            }
        }
    }
    __syncthreads();

    const float again = exp2_int(was - e);  // kept codes' steps in the new scale
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int vec = tid + i * kThreads;
        kv8_u32x4 out = *reinterpret_cast<const kv8_u32x4*>(codes + vec * 16);
        if (!whole) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t m = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    // the cell of byte k of word w
                    const int c = which == 0 ? vec % kBlk : vec % 2 * 16 + w * 4 + k;
                    uint32_t y = out[w] >> (8 * k);
                    if (c < c0 || c >= c1) y = old[i][w] >> (8 * k);
                    if (c < c0) y = (uint32_t)(int)rintf((float)(int8_t)(y & 0xff) * again);
                    m |= (y & 0xff) << (8 * k);
                }
                out[w] = m;
            }
        }
        *reinterpret_cast<kv8_u32x4*>(block + vec * 16) = out;
    }
    if (tid == 0) *exp_p = (int8_t)e;
}

template <int D>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(Kv8RowsArgs a) {
    constexpr int kChunks = kBlk * D / 8 / kThreads;
    constexpr int kVecs = kBlk * D / 16 / kThreads;
    __shared__ __align__(16) uint8_t codes[kBlk * D];
    const int tid = threadIdx.x, s = blockIdx.z, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const Span r = span_of(a, s);
    const int64_t b64 = r.lo / kBlk + blockIdx.x;
    if (r.lo >= r.hi || b64 * kBlk >= r.hi) return;
    const int64_t cell0 = b64 * kBlk;
    const Kv8Tensor& t = a.t[which];
    int64_t at, e_at;
    block_at(a.pages, t.nb, t.e_nb, s, (int)b64, at, e_at);
    const char* block = t.codes + at + (int64_t)head * t.nb[1];
    const float step = exp2_int(clamp_exp(t.exps[e_at + (int64_t)head * t.e_nb[1]]));
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
        *reinterpret_cast<kv8_u32x4*>(codes + (tid + i * kThreads) * 16) =
            *reinterpret_cast<const kv8_u32x4*>(block + (tid + i * kThreads) * 16);
    __syncthreads();
    char* rows = a.rows[which] + (int64_t)head * a.r_nb2[which] + (int64_t)s * a.r_nb3[which];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int id = tid + i * kThreads, c = id / (D / 8), d = id % (D / 8) * 8;
        const int64_t cell = cell0 + c;
        if (cell < r.lo || cell >= r.hi) continue;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint8_t u = which == 0 ? codes[d / 16 * (kBlk * 16) + c * 16 + d % 16 + k] : codes[(d + k) * kBlk + c];
            x[k] = (float)(int8_t)u * step;
        }
        char* p = rows + (cell - r.first) * a.r_nb1[which];
        if (a.f16[which]) {
            kv8_f16x8 h;
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = (_Float16)fminf(fmaxf(x[k], -65504.0f), 65504.0f);
            *reinterpret_cast<kv8_f16x8*>(p + d * 2) = h;
        } else {
            *reinterpret_cast<kv8_f32x4*>(p + d * 4) = kv8_f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<kv8_f32x4*>(p + d * 4 + 16) = kv8_f32x4{x[4], x[5], x[6], x[7]};
        }
    }
}

// Blocks that n rows may touch, wherever they begin.
dim3 rows_grid(const Kv8RowsArgs& a) {
    return dim3((unsigned)((a.n_rows + 2 * kBlk - 2) / kBlk), (unsigned)(2 * a.Hkv), (unsigned)a.S);
}

}  // namespace

hipError_t launch_kv8_write(const Kv8RowsArgs& a, hipStream_t stream) {
    if (a.n_rows == 0 || a.S == 0 || a.Hkv == 0) return hipSuccess;
    if (a.D == 128)
        hipLaunchKernelGGL(kv8_write_kernel<128>, rows_grid(a), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(kv8_write_kernel<256>, rows_grid(a), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8RowsArgs& a, hipStream_t stream) {
    if (a.n_rows == 0 || a.S == 0 || a.Hkv == 0) return hipSuccess;
    if (a.D == 128)
        hipLaunchKernelGGL(kv8_read_kernel<128>, rows_grid(a), dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(kv8_read_kernel<256>, rows_grid(a), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sixi
