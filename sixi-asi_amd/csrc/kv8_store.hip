// kv8_store.hip -- rows into the 8-bit cache and back (include/sixi_kv8.h).
//
// One work-group per (stream, head, K or V, block of 32 cells).  A block's scale is a power of two:
//   e = min { e : max |x| <= 127 * 2^e },  code = rne(x * 2^-e),
// so multiplying by 2^-e is exact and the code is the value's nearest multiple whoever forms it.  A
// block that keeps cells in front of the new rows takes e' = max(e, its own) and shifts the kept codes
// by e' - e with one more rounding; its own exponent never falls until the block is begun anew.
//
// Bound by HBM: rows in once, codes out once; a block that is only partly written is read first (4 or
// 8 KiB), which is what a step that appends one token costs.  Codes pass through LDS as rows of D + 16 bytes:
// written and read there in pieces of 8 bytes (rows), 16 (K: a cell's 16 dims) and 4 (V: a cell's 4 dims, turned
// 4 x 4 in registers into 4 dims' cells), all without bank conflicts, so that every access to the cache is 16
// bytes and a whole block leaves as one piece.  (With V's bytes scattered into LDS one by one a chunk of 2048
// rows of 256 took 13 us instead of 8, and its read-back 13 instead of 5.)
//
// Measured: 2048 f16 rows of 4 heads of 256 dims 8.2 us (13 MB in and out, 1.5 TB/s: four work-groups a CU, one round
// of loads, reductions and stores), read back 5.5 us; a token of 32 streams 6.4 us, read back 4.0: launch and two
// dependent loads.
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

// A work-group's place.
struct Site {
    Span r;
    int64_t cell0;
    int c0, c1;  // the rows' cells in the block
    char* block;
    int8_t* exp;
    bool any;
};
__device__ __forceinline__ Site site_of(const Kv8RowsArgs& a, int s, int which, int head) {
    Site x;
    x.r = span_of(a, s);
    const int64_t b = x.r.lo / kBlk + blockIdx.x;
    x.cell0 = b * kBlk;
    x.any = x.r.lo < x.r.hi && x.cell0 < x.r.hi;
    if (!x.any) return x;
    x.c0 = x.r.lo > x.cell0 ? (int)(x.r.lo - x.cell0) : 0;
    x.c1 = x.r.hi < x.cell0 + kBlk ? (int)(x.r.hi - x.cell0) : kBlk;
    const Kv8Tensor& t = a.t[which];
    int64_t at, e_at;
    block_at(a.pages, t.nb, t.e_nb, s, (int)b, at, e_at);
    x.block = t.codes + at + (int64_t)head * t.nb[1];
    x.exp = t.exps + e_at + (int64_t)head * t.e_nb[1];
    return x;
}

// Four words of four bytes, turned: byte i of word k becomes byte k of word i.
__device__ __forceinline__ void turn4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Unit u of a block: four 16-byte pieces of the cache.  K: pieces u, u + U, ..; V: 16 cells (half u % 2) of the
// dims 4 (u / 2) .. + 3.
template <int D>
struct Unit {
    static constexpr int U = kBlk * D / 64, kRow = D + 16;  // units of a block; bytes of a row in LDS
    __device__ __forceinline__ static int piece(int which, int u, int k) { return which == 0 ? u + k * U : (u / 2 * 4 + k) * 2 + u % 2; }
    // out of rows of codes, and into them
    __device__ __forceinline__ static void gather(const uint8_t* rows, int which, int u, kv8_u32x4 (&x)[4]) {
        if (which == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = piece(0, u, k);
                x[k] = *reinterpret_cast<const kv8_u32x4*>(rows + p % kBlk * kRow + p / kBlk * 16);
            }
        } else {
            const uint8_t* at = rows + u % 2 * 16 * kRow + u / 2 * 4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = *reinterpret_cast<const uint32_t*>(at + (4 * c + k) * kRow);
                turn4(w);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k][c] = w[k];
            }
        }
    }
    __device__ __forceinline__ static void scatter(uint8_t* rows, int which, int u, const kv8_u32x4 (&x)[4]) {
        if (which == 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int p = piece(0, u, k);
                *reinterpret_cast<kv8_u32x4*>(rows + p % kBlk * kRow + p / kBlk * 16) = x[k];
            }
        } else {
            uint8_t* at = rows + u % 2 * 16 * kRow + u / 2 * 4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = x[k][c];
                turn4(w);
#pragma unroll
                for (int k = 0; k < 4; ++k) *reinterpret_cast<uint32_t*>(at + (4 * c + k) * kRow) = w[k];
            }
        }
    }
};

template <int D>
__global__ __launch_bounds__(kThreads) void kv8_write_kernel(Kv8RowsArgs a) {
    typedef Unit<D> Un;
    constexpr int kChunks = kBlk * D / 8 / kThreads;   // 8-element pieces of rows per thread
    __shared__ __align__(16) uint8_t codes[kBlk * Un::kRow];
    __shared__ float tops[kThreads / 64];
    const int tid = threadIdx.x, s = blockIdx.z, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const Site x = site_of(a, s, which, head);
    if (!x.any) return;
    const bool whole = x.c0 == 0 && x.c1 == kBlk;
    kv8_u32x4 old[4];
    if (!whole && tid < Un::U) {
#pragma unroll
        for (int k = 0; k < 4; ++k) old[k] = *reinterpret_cast<const kv8_u32x4*>(x.block + Un::piece(which, tid, k) * 16);
    }
    const int was = x.c0 > 0 ? clamp_exp(*x.exp) : SIXI_KV8_EXP_MIN;

    const char* rows = a.rows[which] + (int64_t)head * a.r_nb2[which] + (int64_t)s * a.r_nb3[which];
    float v[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int id = tid + i * kThreads, c = id / (D / 8), d8 = id % (D / 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        if (c >= x.c0 && c < x.c1) {
            const int64_t row = x.cell0 + c - x.r.first;
            load8(rows + row * a.r_nb1[which] + (int64_t)d8 * (a.f16[which] ? 16 : 32), a.f16[which] != 0, v[i]);
        }
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float m = fabsf(v[i][e]);
            top = fmaxf(top, m < __builtin_huge_valf() ? m : 0.0f);  // finite values only (NaN compares false)
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
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            lo |= (uint32_t)(code_of(v[i][k], inv) & 0xff) << (8 * k);
            hi |= (uint32_t)(code_of(v[i][4 + k], inv) & 0xff) << (8 * k);
        }
        *reinterpret_cast<kv8_u32x2*>(codes + c * Un::kRow + d) = kv8_u32x2{lo, hi};
    }
    __syncthreads();
    if (tid == 0) *x.exp = (int8_t)e;
    if (tid >= Un::U) return;

    kv8_u32x4 out[4];
    Un::gather(codes, which, tid, out);
    if (!whole) {
        // bytes of four cells from b on that lie below cell c
        auto below = [](int c, int b) { return (uint32_t)((1ull << (8 * min(max(c - b, 0), 4))) - 1); };
        const bool grown = e > was;             // the kept codes' scale
        const float again = exp2_int(was - e);  // their steps in the new one
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int piece = Un::piece(which, tid, k), cell = piece % kBlk;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int b = piece % 2 * 16 + 4 * w;
                const uint32_t kept = which == 0 ? (cell < x.c0 ? ~0u : 0u) : below(x.c0, b);
                const uint32_t fresh = (which == 0 ? (cell < x.c1 ? ~0u : 0u) : below(x.c1, b)) & ~kept;
                uint32_t y = old[k][w];
                if (grown) {
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        m |= (uint32_t)((int)rintf((float)(int8_t)(y >> (8 * i)) * again) & 0xff) << (8 * i);
                    y = (m & kept) | (y & ~kept);
                }
                out[k][w] = (out[k][w] & fresh) | (y & ~fresh);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<kv8_u32x4*>(x.block + Un::piece(which, tid, k) * 16) = out[k];
}

template <int D>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(Kv8RowsArgs a) {
    typedef Unit<D> Un;
    constexpr int kChunks = kBlk * D / 8 / kThreads;
    __shared__ __align__(16) uint8_t codes[kBlk * Un::kRow];
    const int tid = threadIdx.x, s = blockIdx.z, which = blockIdx.y & 1, head = blockIdx.y >> 1;
    const Site x = site_of(a, s, which, head);
    if (!x.any) return;
    const float step = exp2_int(clamp_exp(*x.exp));
    if (tid < Un::U) {
        kv8_u32x4 in[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) in[k] = *reinterpret_cast<const kv8_u32x4*>(x.block + Un::piece(which, tid, k) * 16);
        Un::scatter(codes, which, tid, in);
    }
    __syncthreads();
    char* rows = a.rows[which] + (int64_t)head * a.r_nb2[which] + (int64_t)s * a.r_nb3[which];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const int id = tid + i * kThreads, c = id / (D / 8), d = id % (D / 8) * 8;
        if (c < x.c0 || c >= x.c1) continue;
        const kv8_u32x2 w = *reinterpret_cast<const kv8_u32x2*>(codes + c * Un::kRow + d);
        float v[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = (float)(int8_t)(w[0] >> (8 * k)) * step;
            v[4 + k] = (float)(int8_t)(w[1] >> (8 * k)) * step;
        }
        char* p = rows + (x.cell0 + c - x.r.first) * a.r_nb1[which];
        if (a.f16[which]) {
            kv8_f16x8 h;
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = (_Float16)fminf(fmaxf(v[k], -65504.0f), 65504.0f);
            *reinterpret_cast<kv8_f16x8*>(p + d * 2) = h;
        } else {
            *reinterpret_cast<kv8_f32x4*>(p + d * 4) = kv8_f32x4{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<kv8_f32x4*>(p + d * 4 + 16) = kv8_f32x4{v[4], v[5], v[6], v[7]};
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
