// rope.hip -- rotary positions of Q and K (include/sixi_rope.h).
//
// A row's angles are the same for every head: a work-group takes one row (or a share of its heads, where
// rows are few), forms the n_rot/2 pairs of cos and sin once, in LDS, and turns head after head with them.
// An angle is reduced in 64 bits, in turns: pos * (f / 2 pi), less its nearest whole number, is exact to
// 2^-52 of the turns passed; cos and sin of what is left run in f32.  (An f32 product is off by 2^-24 of
// the angle: 5e-3 radians at position 180000.)
//
// 8 consecutive elements per lane, D/8 lanes a head row: 16 or 32 bytes of loads and stores per lane.  The
// partner of an element in the half layout sits n_rot/16 lanes away, in the same register; interleaved
// pairs lie within a lane.  The norm's sum of squares is a sum over the row's lanes.  Every element is read
// by the lane that writes it, so the output may be the input.  HBM-bound: rows in and out once: 2048 f16 rows
// of 28 heads of 128 dims 9.4 us (29 MB, 3.1 TB/s); a token 4 us, which is a launch, a length and its rows.
#include <hip/hip_runtime.h>

#include "rope_internal.hpp"

namespace sixi {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;

// LPR lanes hold a head row (the smallest power of two with 8 * LPR >= D).
template <int LPR>
__global__ __launch_bounds__(kThreads) void qk_rope_kernel(RopeArgs a) {
    __shared__ float cs[kMaxPairs], sn[kMaxPairs];
    const int j = blockIdx.x, s = blockIdx.z;
    const int tid = threadIdx.x, half = a.n_rot / 2;
    const int sub = tid % LPR, d0 = sub * 8;
    const bool in_row = d0 < a.D, turned = d0 < a.n_rot;
    const int heads = a.t[0].heads + a.t[1].heads, per = kThreads / LPR;
    // a head's elements of this lane; the first ones are asked for before the angles are formed
    float x[8];
    auto load = [&](int hh) {
        const int w = hh < a.t[0].heads ? 0 : 1, head = w ? hh - a.t[0].heads : hh;
        const RopeTensor& t = a.t[w];
        if (hh < heads && in_row) {
            const char* p = t.in + (int64_t)head * t.i_nb1 + (int64_t)j * t.i_nb2 + (int64_t)s * t.i_nb3;
            if (t.in_f16) {
                const f16x8 v = *reinterpret_cast<const f16x8*>(p + d0 * 2);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
            } else {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(p + d0 * 4), hi = *reinterpret_cast<const f32x4*>(p + d0 * 4 + 16);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = lo[e];
                    x[4 + e] = hi[e];
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        }
    };
    int h0 = blockIdx.y * per;
    load(h0 + tid / LPR);
    if (a.q_len && j >= a.q_len[s]) return;
    if (tid < half) {
        const int64_t at = a.pos ? (int64_t)a.pos[(int64_t)s * a.pos_stride + j] : (int64_t)(a.kv_len ? a.kv_len[s] : 0) + j;
        const double turns = (double)at * (a.freqs[tid] * 0.15915494309189535);  // 1 / (2 pi)
        const float part = (float)(turns - rint(turns));
        float c, y;
        sincospif(2.0f * part, &y, &c);
        cs[tid] = c * a.mscale;
        sn[tid] = (a.inverse ? -y : y) * a.mscale;
    }
    __syncthreads();
    float c[8], y[8];  // per element: its pair's cos, and its pair's sin with the sign of the partner's term
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        c[e] = 1.0f;
        y[e] = 0.0f;
        if (turned) {
            const int d = d0 + e, pair = a.interleaved ? d / 2 : d < half ? d : d - half;
            const bool first = a.interleaved ? (e & 1) == 0 : d < half;
            c[e] = cs[pair];
            y[e] = first ? -sn[pair] : sn[pair];
        }
    }
    const int shift = half / 8, partner = !turned ? tid : d0 < half ? tid + shift : tid - shift;
    while (true) {
        const int hh = h0 + tid / LPR;
        const int w = hh < a.t[0].heads ? 0 : 1, head = w ? hh - a.t[0].heads : hh;
        const RopeTensor& t = a.t[w];
        const bool on = hh < heads && in_row;
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = x[e];
        h0 += gridDim.y * per;
        if (h0 < heads) load(h0 + tid / LPR);
        if (a.t[0].norm) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(r[e], r[e], ss);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
            const float f = 1.0f / sqrtf(ss / (float)a.D + a.eps);
            if (on) {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(t.norm + d0), hi = *reinterpret_cast<const f32x4*>(t.norm + d0 + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    r[e] = r[e] * f * lo[e];
                    r[4 + e] = r[4 + e] * f * hi[e];
                }
            }
        }
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float other = a.interleaved ? r[e ^ 1] : __shfl(r[e], partner & 63, 64);
            o[e] = turned ? fmaf(r[e], c[e], other * y[e]) : r[e];
        }
        if (on) {
            char* p = t.out + (int64_t)head * t.o_nb1 + (int64_t)j * t.o_nb2 + (int64_t)s * t.o_nb3;
            if (t.out_f16) {
                f16x8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (_Float16)o[e];
                *reinterpret_cast<f16x8*>(p + d0 * 2) = v;
            } else {
                *reinterpret_cast<f32x4*>(p + d0 * 4) = f32x4{o[0], o[1], o[2], o[3]};
                *reinterpret_cast<f32x4*>(p + d0 * 4 + 16) = f32x4{o[4], o[5], o[6], o[7]};
            }
        }
        if (h0 >= heads) return;
    }
}

}  // namespace

hipError_t launch_qk_rope(const RopeArgs& a, hipStream_t stream) {
    const int heads = a.t[0].heads + a.t[1].heads;
    if (a.n_rows == 0 || a.S == 0 || heads == 0) return hipSuccess;
    // few rows: a work-group for each group of heads that its lanes hold at once (their angles formed again
    // cost less than waiting for one group after another: a token of 28 heads 7.8 us and 4.0 so)
    const int per = kThreads / (a.D > 128 ? 32 : a.D > 64 ? 16 : 8), passes = (heads + per - 1) / per;
    const dim3 grid((unsigned)a.n_rows, (int64_t)a.n_rows * a.S <= 1024 ? (unsigned)passes : 1u, (unsigned)a.S);
    if (a.D > 128)
        hipLaunchKernelGGL(qk_rope_kernel<32>, grid, dim3(kThreads), 0, stream, a);
    else if (a.D > 64)
        hipLaunchKernelGGL(qk_rope_kernel<16>, grid, dim3(kThreads), 0, stream, a);
    else
        hipLaunchKernelGGL(qk_rope_kernel<8>, grid, dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sixi
