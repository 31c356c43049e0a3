// draft_verify.hip -- which drafted tokens stay, and the token behind them (include/sixi_draft.h).
//
// Three launches, each a function of its inputs alone (no atomics, sums in a fixed order):
//   rows    every row's chunks of 4096 logits: largest, its token, sum of exp((l - max) / T)
//   draw    per stream, the accept chain from those sums (a few hundred numbers, formed again by each
//           work-group), then the chunk's share of the row that the next token is drawn from
//   find    the chunk and the token at which the running sum passes u_next * total
// Bound by HBM: the logits once (the row that is drawn from a second time, out of the caches).  Sums and
// exponentials run in 64 bits: a token is found between neighbours of a running sum over the whole
// vocabulary, where 1e-7 of the total spans many of them.  2^x is formed from its whole part and a
// polynomial of degree 11 in the rest (the Taylor terms of exp to 1e-13 on [-0.35, 0.35]): about 16 f64
// instructions, hidden behind the loads.
#include <hip/hip_runtime.h>

#include "draft_internal.hpp"
#include "sixi_draft.h"

namespace sixi {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = kDraftChunk / kThreads;  // logits per thread

// exp(x) for x <= 0 (0 below -700)
__device__ __forceinline__ double exp_neg(double x) {
    if (!(x > -700.0)) return 0.0;
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, x);  // (off by 2.4e-17 n: below 3e-14 of the result)
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

// exp((l - top) / T): 1 at the top itself (also where both are infinite), 0 for -inf and NaN
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    return l == top ? 1.0 : exp_neg(((double)l - (double)top) * inv_t);
}

__device__ __forceinline__ float load1(const char* p, int type) {
    if (type == SIXI_TYPE_F32) return *reinterpret_cast<const float*>(p);
    const uint16_t h = *reinterpret_cast<const uint16_t*>(p);
    if (type == SIXI_TYPE_F16) return (float)__builtin_bit_cast(_Float16, h);
    return __builtin_bit_cast(float, (uint32_t)h << 16);
}
__device__ __forceinline__ int bytes_of(int type) { return type == SIXI_TYPE_F32 ? 4 : 2; }

__device__ __forceinline__ float heat_of(const DraftArgs& a, int s) { return a.temperature ? a.temperature[s] : 1.0f; }
__device__ __forceinline__ int rows_of(const DraftArgs& a, int s) {
    return a.q_len ? min(max(a.q_len[s], 0), a.n_rows) : a.n_rows;
}

// The larger of two (logit, token) pairs, the lower token of equals; NaN never wins.
__device__ __forceinline__ void take_top(float& top, int& at, float top2, int at2) {
    if (top2 > top || (top2 == top && at2 < at)) {
        top = top2;
        at = at2;
    }
}

__global__ __launch_bounds__(kThreads) void draft_rows_kernel(DraftArgs a) {
    __shared__ float tops[kThreads / 64];
    __shared__ int ats[kThreads / 64];
    __shared__ double sums[kThreads / 64];
    const int chunk = blockIdx.x, j = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    if (j >= rows_of(a, s)) return;
    const int es = bytes_of(a.l_type);
    const char* row = a.logits + (int64_t)j * a.l_nb1 + (int64_t)s * a.l_nb2;
    float x[kPer];
    float top = -__builtin_huge_valf();
    int at = a.V;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int v = chunk * kDraftChunk + i * kThreads + tid;
        x[i] = v < a.V ? load1(row + (int64_t)v * es, a.l_type) : -__builtin_huge_valf();
        if (v < a.V) take_top(top, at, x[i], v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) take_top(top, at, __shfl_xor(top, o, 64), __shfl_xor(at, o, 64));
    if (tid % 64 == 0) {
        tops[tid / 64] = top;
        ats[tid / 64] = at;
    }
    __syncthreads();
    top = tops[0];
    at = ats[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) take_top(top, at, tops[w], ats[w]);
    const float heat = heat_of(a, s);
    double sum = 0.0;
    if (heat > 0.0f && top > -__builtin_huge_valf()) {
        const double inv_t = 1.0 / (double)heat;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += weight(x[i], top, inv_t);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (tid % 64 == 0) sums[tid / 64] = sum;
    __syncthreads();
    if (tid == 0) {
        DraftPart& p = a.parts[((int64_t)s * a.n_rows + j) * a.chunks + chunk];
        p.sum = ((sums[0] + sums[1]) + sums[2]) + sums[3];
        p.top = top;
        p.at = at;
    }
}

// What a stream's rows come to, formed by every work-group that needs it.
struct Verdict {
    int row;        // the row that the next token is drawn from
    int d;          // its drafted token (V: none in range); -1 behind the last one
    float top;      // of that row
    int at;
    double inv_z;   // 1 / its sum of weights
    double inv_t;   // 0: greedy
};

constexpr int kGroup = 16;  // lanes that sum a row's chunks

// A row's largest logit and sum of weights, by the 16 lanes of a group (every lane gets them).
__device__ __forceinline__ void row_sum(const DraftArgs& a, int s, int j, double inv_t, float& top, int& at, double& z) {
    const int lane = threadIdx.x % kGroup;
    const DraftPart* parts = a.parts + ((int64_t)s * a.n_rows + j) * a.chunks;
    top = -__builtin_huge_valf();
    at = a.V;
    for (int c = lane; c < a.chunks; c += kGroup) take_top(top, at, parts[c].top, parts[c].at);
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) take_top(top, at, __shfl_xor(top, o, 64), __shfl_xor(at, o, 64));
    z = 0.0;
    for (int c = lane; c < a.chunks; c += kGroup) z += parts[c].sum * weight(parts[c].top, top, inv_t);
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
}

// Each group of 16 lanes judges rows of its own; `stop` (LDS) is then the first whose token goes, or the
// last row.  Every thread of the work-group calls this.
__device__ __forceinline__ Verdict decide(const DraftArgs& a, int s, int rows, int* stop) {
    const float heat = heat_of(a, s);
    const bool greedy = !(heat > 0.0f);
    Verdict v{};
    v.inv_t = greedy ? 0.0 : 1.0 / (double)heat;
    if (threadIdx.x == 0) *stop = rows - 1;
    __syncthreads();
    for (int j = threadIdx.x / kGroup; j < rows - 1; j += kThreads / kGroup) {
        float top;
        int at;
        double z, p = 0.0, q = 1.0;
        const int d = a.draft[(int64_t)s * a.draft_stride + j];
        const bool known = d >= 0 && d < a.V;
        float l = 0.0f;
        if (known) {
            l = load1(a.logits + (int64_t)j * a.l_nb1 + (int64_t)s * a.l_nb2 + (int64_t)d * bytes_of(a.l_type), a.l_type);
            if (a.probs)
                q = load1(a.probs + (int64_t)j * a.p_nb1 + (int64_t)s * a.p_nb2 + (int64_t)d * bytes_of(a.p_type), a.p_type);
        }
        row_sum(a, s, j, v.inv_t, top, at, z);
        if (known) p = greedy ? (d == at ? 1.0 : 0.0) : z > 0.0 ? weight(l, top, v.inv_t) / z : 0.0;
        if (!((double)a.u[(int64_t)s * a.u_stride + j] * q < p) && threadIdx.x % kGroup == 0) atomicMin(stop, j);
    }
    __syncthreads();
    v.row = *stop;
    double z;
    row_sum(a, s, v.row, v.inv_t, v.top, v.at, z);
    v.inv_z = z > 0.0 ? 1.0 / z : 0.0;
    v.d = -1;
    if (v.row < rows - 1) {
        v.d = a.draft[(int64_t)s * a.draft_stride + v.row];
        if (v.d < 0 || v.d > a.V) v.d = a.V;
    }
    return v;
}

// Weights of token t for the draw, and of p.
__device__ __forceinline__ void weights_at(const DraftArgs& a, int s, const Verdict& v, int t, double& w, double& p) {
    p = 0.0;
    if (v.inv_t == 0.0) {
        p = t == v.at ? 1.0 : 0.0;
    } else if (v.top > -__builtin_huge_valf()) {
        p = weight(load1(a.logits + (int64_t)v.row * a.l_nb1 + (int64_t)s * a.l_nb2 + (int64_t)t * bytes_of(a.l_type), a.l_type), v.top,
                   v.inv_t) * v.inv_z;
    }
    w = p;
    if (v.d >= 0) {
        double q = t == v.d ? 1.0 : 0.0;
        if (a.probs)
            q = load1(a.probs + (int64_t)v.row * a.p_nb1 + (int64_t)s * a.p_nb2 + (int64_t)t * bytes_of(a.p_type), a.p_type);
        w = p - q > 0.0 ? p - q : 0.0;
    }
}

__global__ __launch_bounds__(kThreads) void draft_draw_kernel(DraftArgs a) {
    __shared__ double ws[kThreads / 64], ps[kThreads / 64];
    __shared__ int lws[kThreads / 64], lps[kThreads / 64], stop;
    const int chunk = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int rows = rows_of(a, s);
    if (rows == 0) return;
    const Verdict v = decide(a, s, rows, &stop);
    if (chunk == 0 && tid == 0) a.keep[s] = v.row + 1;
    double w = 0.0, p = 0.0;
    int last_w = -1, last_p = -1;
    for (int i = 0; i < kPer; ++i) {
        const int t = chunk * kDraftChunk + i * kThreads + tid;
        if (t >= a.V) break;
        double tw, tp;
        weights_at(a, s, v, t, tw, tp);
        w += tw;
        p += tp;
        if (tw > 0.0) last_w = t;
        if (tp > 0.0) last_p = t;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        w += __shfl_xor(w, o, 64);
        p += __shfl_xor(p, o, 64);
        last_w = max(last_w, __shfl_xor(last_w, o, 64));
        last_p = max(last_p, __shfl_xor(last_p, o, 64));
    }
    if (tid % 64 == 0) {
        ws[tid / 64] = w;
        ps[tid / 64] = p;
        lws[tid / 64] = last_w;
        lps[tid / 64] = last_p;
    }
    __syncthreads();
    if (tid == 0) {
        DraftDraw& d = a.draws[(int64_t)s * a.chunks + chunk];
        d.w = ((ws[0] + ws[1]) + ws[2]) + ws[3];
        d.p = ((ps[0] + ps[1]) + ps[2]) + ps[3];
        d.last_w = max(max(lws[0], lws[1]), max(lws[2], lws[3]));
        d.last_p = max(max(lps[0], lps[1]), max(lps[2], lps[3]));
    }
}

__global__ __launch_bounds__(kThreads) void draft_find_kernel(DraftArgs a) {
    __shared__ double sums[kThreads];
    __shared__ int stop, first, found;
    const int s = blockIdx.x, tid = threadIdx.x;
    const int rows = rows_of(a, s);
    if (rows == 0) {
        if (tid == 0) {
            a.keep[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    const Verdict v = decide(a, s, rows, &stop);
    // the chunk: every thread walks the same few dozen sums
    const DraftDraw* d = a.draws + (int64_t)s * a.chunks;
    double total = 0.0;
    for (int c = 0; c < a.chunks; ++c) total += d[c].w;
    const bool from_w = total > 0.0;
    if (!from_w) {
        total = 0.0;
        for (int c = 0; c < a.chunks; ++c) total += d[c].p;
        if (!(total > 0.0)) {
            if (tid == 0) a.token[s] = -1;
            return;
        }
    }
    const double mark = (double)a.u_next[s] * total;
    // the first chunk whose end is past the mark; where the sums' rounding (or u_next = 1) leaves none, the
    // last one with a weight
    double before = 0.0, sum = 0.0;
    int chunk = 0, last = -1;
    for (int c = 0; c < a.chunks; ++c) {
        const int tail = from_w ? d[c].last_w : d[c].last_p;
        if (tail < 0) continue;
        before = sum;
        chunk = c;
        last = tail;
        sum += from_w ? d[c].w : d[c].p;
        if (sum > mark) break;
    }
    // 16 consecutive tokens per thread, then the running sum over the threads (log steps: the same sums
    // in every call)
    const int t0 = chunk * kDraftChunk + tid * kPer;
    double mine = 0.0;
    for (int i = 0; i < kPer; ++i) {
        if (t0 + i >= a.V) break;
        double w, p;
        weights_at(a, s, v, t0 + i, w, p);
        mine += from_w ? w : p;
    }
    sums[tid] = mine;
    if (tid == 0) {
        first = kThreads;
        found = last;
    }
    __syncthreads();
#pragma unroll
    for (int o = 1; o < kThreads; o <<= 1) {
        const double x = tid >= o ? sums[tid - o] : 0.0;
        __syncthreads();
        sums[tid] += x;
        __syncthreads();
    }
    if (mine > 0.0 && before + sums[tid] > mark) atomicMin(&first, tid);
    __syncthreads();
    if (tid == first) {
        double run = before + (tid > 0 ? sums[tid - 1] : 0.0);
        int at = -1;
        for (int i = 0; i < kPer; ++i) {
            if (t0 + i >= a.V) break;
            double w, p;
            weights_at(a, s, v, t0 + i, w, p);
            const double x = from_w ? w : p;
            if (!(x > 0.0)) continue;
            run += x;
            at = t0 + i;
            if (run > mark) break;
        }
        found = at;
    }
    __syncthreads();
    if (tid == 0) a.token[s] = found;
}

}  // namespace

hipError_t launch_draft_verify(const DraftArgs& a, hipStream_t stream) {
    if (a.S == 0) return hipSuccess;
    hipLaunchKernelGGL(draft_rows_kernel, dim3((unsigned)a.chunks, (unsigned)a.n_rows, (unsigned)a.S), dim3(kThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(draft_draw_kernel, dim3((unsigned)a.chunks, (unsigned)a.S), dim3(kThreads), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(draft_find_kernel, dim3((unsigned)a.S), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace sixi
