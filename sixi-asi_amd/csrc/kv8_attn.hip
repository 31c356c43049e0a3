// kv8_attn.hip -- attention over the 8-bit cache (include/sixi_kv8.h).
//
// One pass over the cells with the running maximum and sum of a softmax.  A group's rows (row j of the
// G heads that share a kv-head; row index r = j * G + h) are taken 32 at a time as the columns of
//   S^T[cell, row] = K Q^T      O^T[dim, row] += V^T P^T
// on v_mfma_f32_32x32x16_f16, a block of 32 cells per step.  Both left operands come from the cache as
// it lies in memory: 16 bytes per lane, 1 KiB per wave.  Codes become f16 exactly (|code| <= 127), the
// scales are powers of two and never meet an element:
//   t = scale log2(e) 2^ek (q . k) + ev        the exponent of (weight * 2^ev)
//   P' = 2^(t - m)                              m the running maximum of t (less kHead)
//   O' = sum P' v,   l = sum P' 2^-ev,   o = O' / l
// With ev inside the exponent a block's V scale costs nothing, and the f16 rounding of P' is half a step
// of 11 bits of each weight, down to 2^-24 of the largest contribution whatever the blocks' scales are.
// l is summed from the unrounded weights in f32.
//
// The cell that score register i of a lane holds is ours to choose (any order of K's rows will do):
// lane (n, h) of the 32 x 32 result holds cells 16h .. 16h + 15 of the block in order, which is what the
// lane needs as its half of the next product's right operand.  So P never leaves its lane.
#include "kv8_device.hpp"

namespace sixi {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3e38f;  // below every score: the running maximum of a row that has seen no cell
// The largest weight is 2^kHead, not 1: f16 weights keep 11 bits down to 2^-24 of it.
constexpr float kHead = 10.0f;

// Four int8 codes as f16, exactly: the code + 128 under the exponent of 1024, less 1152.
__device__ __forceinline__ void codes_f16(uint32_t c, f16x2& lo, f16x2& hi) {
    const uint32_t u = c ^ 0x80808080u;
    const f16x2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off;
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off;
}
__device__ __forceinline__ void codes_f16x16(kv8_u32x4 c, kv8_f16x8& a, kv8_f16x8& b) {
    f16x2 p[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) codes_f16(c[i], p[2 * i], p[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[2 * i] = p[i][0];
        a[2 * i + 1] = p[i][1];
        b[2 * i] = p[4 + i][0];
        b[2 * i + 1] = p[4 + i][1];
    }
}

__device__ __forceinline__ f32x16 mfma(kv8_f16x8 a, kv8_f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// What a stream's rows see: rows of the block, cells before it, cells in all.
struct Lens {
    int rows, cached, cells;
};
__device__ __forceinline__ Lens lens_of(const Kv8AttnArgs& a, int s) {
    Lens r;
    r.rows = a.q_len ? min(max(a.q_len[s], 0), a.n_q) : a.n_q;
    r.cached = a.kv_len ? min(max(a.kv_len[s], 0), a.n_kv - r.rows) : a.n_kv - r.rows;
    r.cells = r.cached + r.rows;  // (without kv_len: all n_kv)
    return r;
}

// Blocks [first, last) of piece `i` of `n` of a stream.
__device__ __forceinline__ void piece_of(int cells, int i, int n, int& first, int& last) {
    const int blocks = (cells + kBlk - 1) / kBlk, each = (blocks + n - 1) / n;
    first = min(i * each, blocks);
    last = min(first + each, blocks);
}

__device__ __forceinline__ float* slot_of(const Kv8AttnArgs& a, int s, int g, int tile, int piece) {
    return a.part + ((((int64_t)s * a.Hkv + g) * a.n_tiles + tile) * a.n_split + piece) * (32 * (int64_t)a.D + 64);
}

__device__ __forceinline__ void store4(const Kv8AttnArgs& a, char* row, int d, kv8_f32x4 x) {
    if (a.o_f16) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        f16x4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = (_Float16)x[i];
        *reinterpret_cast<f16x4*>(row + d * 2) = h;
    } else {
        *reinterpret_cast<kv8_f32x4*>(row + d * 4) = x;
    }
}

constexpr int kWaves = 4;

template <int D, bool MASK>
__global__ __launch_bounds__(kWaves * 64, D == 128 ? 2 : 1) void kv8_attn_kernel(Kv8AttnArgs a) {
    constexpr int KC = D / 32;  // 32-dim pieces of a row: K loads, V loads and output tiles
    extern __shared__ __align__(16) float lds[];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int piece = blockIdx.x % a.n_split, tile = blockIdx.x / a.n_split, g = blockIdx.y, s = blockIdx.z;
    const Lens len = lens_of(a, s);
    const int M = len.rows * a.G;
    if (tile * 32 >= M) return;
    int b0, b1;
    piece_of(len.cells, piece, a.n_split, b0, b1);
    if (b0 >= b1 && piece > 0) return;

    // the lane's row: its query, and the last cell that it sees
    const int r = tile * 32 + n;
    const bool live = r < M;
    const int j = live ? r / a.G : 0, head = live ? g * a.G + r % a.G : g * a.G;
    const int last = a.mode == SIXI_MASK_BLOCK_CAUSAL ? len.cached + j : len.cells - 1;
    const int sees = a.mode == SIXI_MASK_BLOCK_CAUSAL ? len.cached + tile * 32 / a.G : len.cells - 1;  // by every row
    // cells behind the last that any row of the tile sees are not read
    const int jl = (min(tile * 32 + 32, M) - 1) / a.G;
    const int reach = a.mode == SIXI_MASK_BLOCK_CAUSAL ? len.cached + jl + 1 : len.cells;
    b1 = min(b1, (reach + kBlk - 1) / kBlk);
    kv8_f16x8 q[KC][2];
    {
        const char* p = a.q + (int64_t)j * a.q_nb1 + (int64_t)head * a.q_nb2 + (int64_t)s * a.q_nb3;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = (2 * c + h) * 16 + 8 * u;
                kv8_f16x8 x;
                if (a.q_f16) {
                    x = *reinterpret_cast<const kv8_f16x8*>(p + d * 2);
                } else {
                    const kv8_f32x4 lo = *reinterpret_cast<const kv8_f32x4*>(p + d * 4);
                    const kv8_f32x4 hi = *reinterpret_cast<const kv8_f32x4*>(p + d * 4 + 16);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[i] = (_Float16)lo[i];
                        x[4 + i] = (_Float16)hi[i];
                    }
                }
                const _Float16 sign = (_Float16)(live ? a.q_sign : 0.0f);
                q[c][u] = live ? x * sign : kv8_f16x8{};
            }
    }
    const char* mask = nullptr;
    if (MASK) mask = a.mask + (int64_t)j * a.m_nb1 + (int64_t)s * a.m_nb3;

    f32x16 o[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) o[c] = f32x16{};
    float m = kLowest, l = 0.0f;
    const int k_off = h * (kBlk * 16) + (16 * (n / 4 % 2) + 4 * (n / 8) + n % 4) * 16;
    const int v_off = n * kBlk + h * 16;

    for (int b = b0 + wave; b < b1; b += kWaves) {
        int64_t k_at, ke_at, v_at, ve_at;
        block_at(a.pages, a.k.nb, a.k.e_nb, s, b, k_at, ke_at);
        block_at(a.pages, a.v.nb, a.v.e_nb, s, b, v_at, ve_at);
        const char* kp = a.k.codes + k_at + (int64_t)g * a.k.nb[1];
        const char* vp = a.v.codes + v_at + (int64_t)g * a.v.nb[1];
        kv8_u32x4 kc[KC], vc[KC];
#pragma unroll
        for (int c = 0; c < KC; ++c) kc[c] = *reinterpret_cast<const kv8_u32x4*>(kp + k_off + c * (kBlk * 32));
#pragma unroll
        for (int c = 0; c < KC; ++c) vc[c] = *reinterpret_cast<const kv8_u32x4*>(vp + v_off + c * (kBlk * 32));
        const int ek = clamp_exp(a.k.exps[ke_at + (int64_t)g * a.k.e_nb[1]]);
        const int ev = clamp_exp(a.v.exps[ve_at + (int64_t)g * a.v.e_nb[1]]);

        f32x16 sc = {};
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            kv8_f16x8 x, y;
            codes_f16x16(kc[c], x, y);
            sc = mfma(x, q[c][0], sc);
            sc = mfma(y, q[c][1], sc);
        }
        const float ks = a.scale_log2 * exp2_int(ek), es = (float)ev;
        const int cell0 = b * kBlk + 16 * h;
        float top;
        if (MASK) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float add = -__builtin_huge_valf();
                if (cell0 + i <= last) add = (float)*reinterpret_cast<const _Float16*>(mask + (int64_t)(cell0 + i) * 2);
                sc[i] = fmaf(sc[i], ks, fmaf(add, kLog2e, es));
            }
            top = sc[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
        } else {
            if (b * kBlk + kBlk - 1 > sees) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (cell0 + i > last) sc[i] = -__builtin_huge_valf();
            }
            top = sc[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, sc[i]);
            top = fmaf(top, ks, es);
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float up = fmaxf(m, top - kHead);
        if (__builtin_amdgcn_ballot_w64(up > m)) {
            const float f = __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= f;
#pragma unroll
            for (int c = 0; c < KC; ++c) o[c] *= f;
        }
        const float sub = MASK ? -m : es - m;
        float sum = 0.0f;
        kv8_f16x8 p[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float w = __builtin_amdgcn_exp2f(MASK ? sc[i] + sub : fmaf(sc[i], ks, sub));
            sum += w;
            p[i / 8][i % 8] = (_Float16)w;
        }
        l = fmaf(sum, exp2_int(-ev), l);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            kv8_f16x8 x, y;
            codes_f16x16(vc[c], x, y);
            o[c] = mfma(x, p[0], o[c]);
            o[c] = mfma(y, p[1], o[c]);
        }
    }
    l += __shfl_xor(l, 32, 64);

    // the waves' results into the first one's, two and then one at a time
    for (int half = kWaves / 2; half > 0; half /= 2) {
        float* buf = lds + (wave % half) * (32 * D + 64);
        if (wave >= half && wave < 2 * half) {
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) buf[(c * 16 + i) * 64 + lane] = o[c][i];
            if (h == 0) {
                buf[32 * D + n] = m;
                buf[32 * D + 32 + n] = l;
            }
        }
        __syncthreads();
        if (wave < half) {
            const float m2 = buf[32 * D + n], l2 = buf[32 * D + 32 + n], up = fmaxf(m, m2);
            const float f = __builtin_amdgcn_exp2f(m - up), f2 = __builtin_amdgcn_exp2f(m2 - up);
            m = up;
            l = l * f + l2 * f2;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[c][i] = o[c][i] * f + buf[(c * 16 + i) * 64 + lane] * f2;
        }
        __syncthreads();
    }
    if (wave != 0 || !live) return;
    if (a.n_split == 1) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        char* row = a.out + (int64_t)head * a.o_nb1 + (int64_t)j * a.o_nb2 + (int64_t)s * a.o_nb3;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                store4(a, row, c * 32 + 2 * i + 4 * h,
                       kv8_f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]} * inv);
    } else {
        float* part = slot_of(a, s, g, tile, piece);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<kv8_f32x4*>(part + n * D + c * 32 + 2 * i + 4 * h) =
                    kv8_f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
        if (h == 0) {
            part[32 * D + n] = m;
            part[32 * D + 32 + n] = l;
        }
    }
}

// One work-group per (stream, kv-head, tile): a row's pieces in their order.
template <int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8AttnArgs a) {
    const int tile = blockIdx.x, g = blockIdx.y, s = blockIdx.z;
    const Lens len = lens_of(a, s);
    const int M = len.rows * a.G;
    if (tile * 32 >= M) return;
    const int blocks = (len.cells + kBlk - 1) / kBlk, each = (blocks + a.n_split - 1) / a.n_split;
    const int pieces = each > 0 ? (blocks + each - 1) / each : 1;
    for (int x = threadIdx.x; x < 32 * D / 4; x += blockDim.x) {
        const int n = x / (D / 4), d = x % (D / 4) * 4, r = tile * 32 + n;
        if (r >= M) continue;
        const float* p = slot_of(a, s, g, tile, 0);
        const int64_t stride = 32 * (int64_t)D + 64;
        float m = kLowest;
        for (int i = 0; i < pieces; ++i) m = fmaxf(m, p[i * stride + 32 * D + n]);
        float l = 0.0f;
        kv8_f32x4 o = {};
        for (int i = 0; i < pieces; ++i) {
            const float f = __builtin_amdgcn_exp2f(p[i * stride + 32 * D + n] - m);
            l = fmaf(p[i * stride + 32 * D + 32 + n], f, l);
            o += *reinterpret_cast<const kv8_f32x4*>(p + i * stride + n * D + d) * f;
        }
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const int j = r / a.G, head = g * a.G + r % a.G;
        store4(a, a.out + (int64_t)head * a.o_nb1 + (int64_t)j * a.o_nb2 + (int64_t)s * a.o_nb3, d, o * inv);
    }
}

template <int D>
hipError_t launch(const Kv8AttnArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.n_tiles * a.n_split), (unsigned)a.Hkv, (unsigned)a.S);
    const size_t lds = (size_t)(kWaves / 2) * kv8_slot_floats(D) * sizeof(float);
    if (a.mode == SIXI_MASK_EXPLICIT)
        hipLaunchKernelGGL((kv8_attn_kernel<D, true>), grid, dim3(kWaves * 64), lds, stream, a);
    else
        hipLaunchKernelGGL((kv8_attn_kernel<D, false>), grid, dim3(kWaves * 64), lds, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.n_split == 1) return e;
    hipLaunchKernelGGL(kv8_merge_kernel<D>, dim3((unsigned)a.n_tiles, (unsigned)a.Hkv, (unsigned)a.S), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

// Two rounds of work-groups, in pieces of at least 8 blocks (two steps of a wave).
int kv8_attn_splits(int64_t S, int64_t Hkv, int64_t tiles, int64_t n_kv) {
    const int64_t groups = S * Hkv * tiles, blocks = (n_kv + kBlk - 1) / kBlk;
    int64_t n = (512 + groups - 1) / groups;
    if (n > (blocks + 7) / 8) n = (blocks + 7) / 8;
    return (int)(n < 1 ? 1 : n > 128 ? 128 : n);
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t stream) {
    return a.D == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace sixi
