// draft_verify.hip -- which drafted tokens stay, and the token behind them (include/sixi_draft.h).
//
// Three launches, each a function of its inputs alone (no atomics on sums, every sum in a fixed order):
//   rows    every row's chunks of 4096 logits: largest, its token (where a greedy stream asks for it), sum of
//           exp((l - max) / T)
//   draw    per stream, the accept chain from those sums (a few hundred numbers, formed again by each
//           work-group), then the chunk's share of the row that the next token is drawn from
//   find    the chunk and the token at which the running sum passes u_next * total
// Bound by HBM: the logits once (the row that is drawn from a second time, out of the caches).  Sums and
// exponentials run in 64 bits: a token is found between neighbours of a running sum over the whole
// vocabulary, where 1e-7 of the total spans many of them.  exp is formed from its power of two and a
// polynomial of degree 8 in the rest (Chebyshev interpolation on +-ln(2)/2: off by at most 1.1e-12), about
// 16 f64 instructions, next to the loads.
#include <hip/hip_runtime.h>

#include "draft_internal.hpp"
#include "sixi_draft.h"

namespace sixi {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = kDraftChunk / kThreads;  // logits per thread

// exp(x) for x <= 0 (0 below -700)
__device__ __forceinline__ double exp_neg(double x) {
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -0.6931471805599453, x);  // (off by 2.4e-17 n: below 3e-14 of the result)
    double p = 2.4884309742982776e-05;
    p = fma(p, r, 0.00019915868734151192);
    p = fma(p, r, 0.0013888802102825077);
    p = fma(p, r, 0.00833326609438625);
    p = fma(p, r, 0.041666667037968945);
    p = fma(p, r, 0.1666666689106594);
    p = fma(p, r, 0.4999999999944456);
    p = fma(p, r, 0.9999999999797822);
    p = fma(p, r, 1.0000000000000133);
    return x > -700.0 ? ldexp(p, (int)n) : 0.0;
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

template <int TYPE>
struct Elem {
    static constexpr int bytes = TYPE == SIXI_TYPE_F32 ? 4 : 2, per = 16 / bytes;  // elements of a 16-byte load
};
// 16 bytes of a row from element t on (rows begin at any element's address), -inf past the end
template <int TYPE>
__device__ __forceinline__ void load_vec(const char* row, int t, int V, float* x) {
    constexpr int n = Elem<TYPE>::per;
    if (t + n <= V) {
        if constexpr (TYPE == SIXI_TYPE_F32) {
            typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
            const vec v = *reinterpret_cast<const vec*>(row + (int64_t)t * 4);
#pragma unroll
            for (int i = 0; i < n; ++i) x[i] = v[i];
        } else if constexpr (TYPE == SIXI_TYPE_F16) {
            typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
            const vec v = *reinterpret_cast<const vec*>(row + (int64_t)t * 2);
#pragma unroll
            for (int i = 0; i < n; ++i) x[i] = (float)v[i];
        } else {
            typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
            const vec v = *reinterpret_cast<const vec*>(row + (int64_t)t * 2);
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const uint32_t u = (uint32_t)v[i] << 16;
                x[i] = __uint_as_float(u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < n; ++i) x[i] = t + i < V ? load1(row + (int64_t)(t + i) * Elem<TYPE>::bytes, TYPE) : -__builtin_huge_valf();
    }
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o, 64));
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// A wave takes a quarter of the chunk by itself; the four are joined behind the only barrier.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void draft_rows_kernel(DraftArgs a) {
    constexpr int kVec = Elem<TYPE>::per, kWaves = kThreads / 64;
    __shared__ float tops[kWaves];
    __shared__ int ats[kWaves];
    __shared__ double sums[kWaves];
    const int chunk = blockIdx.x, j = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    if (j >= rows_of(a, s)) return;
    const char* row = a.logits + (int64_t)j * a.l_nb1 + (int64_t)s * a.l_nb2;
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i += kVec) load_vec<TYPE>(row, chunk * kDraftChunk + i * kThreads + tid * kVec, a.V, x + i);
    const float heat = heat_of(a, s);
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) top = fmaxf(top, x[i]);  // (fmaxf passes over NaN)
    top = wave_max(top);
    if (!(top > -__builtin_huge_valf())) top = -__builtin_huge_valf();  // (a wave of NaN)
    int at = a.V;
    double sum = 0.0;
    if (!(heat > 0.0f)) {
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
            if (x[i] == top) at = min(at, chunk * kDraftChunk + i / kVec * kVec * kThreads + tid * kVec + i % kVec);
        if (!(top > -__builtin_huge_valf())) at = a.V;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
    } else if (top > -__builtin_huge_valf()) {
        const double inv_t = 1.0 / (double)heat;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += weight(x[i], top, inv_t);
        sum = wave_sum(sum);
    }
    if (tid % 64 == 0) {
        tops[tid / 64] = top;
        ats[tid / 64] = at;
        sums[tid / 64] = sum;
    }
    __syncthreads();
    if (tid == 0) {
        float best = tops[0];
        int best_at = ats[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) take_top(best, best_at, tops[w], ats[w]);
        double z = 0.0;
        if (heat > 0.0f && best > -__builtin_huge_valf()) {
            const double inv_t = 1.0 / (double)heat;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) z += sums[w] * weight(tops[w], best, inv_t);
        }
        DraftPart& p = a.parts[((int64_t)s * a.n_rows + j) * a.chunks + chunk];
        p.sum = z;
        p.top = best;
        p.at = best_at;
    }
}

constexpr int kGroup = 16;  // lanes that sum a row's chunks

// A row's largest logit and sum of weights, by the 16 lanes of a group (every lane gets them).
__device__ __forceinline__ void row_sum(const DraftArgs& a, int s, int j, double inv_t, float& top, int& at, double& z) {
    const int lane = threadIdx.x % kGroup;
    const DraftPart* parts = a.parts + ((int64_t)s * a.n_rows + j) * a.chunks;
    top = -__builtin_huge_valf();
    at = a.V;
#pragma unroll 4
    for (int c = lane; c < a.chunks; c += kGroup) take_top(top, at, parts[c].top, parts[c].at);
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) take_top(top, at, __shfl_xor(top, o, 64), __shfl_xor(at, o, 64));
    z = 0.0;
#pragma unroll 4
    for (int c = lane; c < a.chunks; c += kGroup) z += parts[c].sum * weight(parts[c].top, top, inv_t);
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
}

// Each group of 16 lanes judges rows of its own; `stop` (LDS) is then the first whose token goes, or the
// last row.  Every thread of the work-group calls this.
__device__ __forceinline__ DraftVerdict decide(const DraftArgs& a, int s, int rows, int* stop) {
    const float heat = heat_of(a, s);
    const bool greedy = !(heat > 0.0f);
    DraftVerdict v{};
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

// Weights of a thread's 16 tokens from t0 on, for the draw and of p (0 past the end).
template <int TYPE>
__device__ __forceinline__ void weights_of(const DraftArgs& a, int s, const DraftVerdict& v, int t0, double (&w)[kPer], double (&p)[kPer]) {
    float x[kPer], q[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        x[i] = -__builtin_huge_valf();
        q[i] = 0.0f;
    }
    const bool hot = v.inv_t != 0.0 && v.top > -__builtin_huge_valf();
    if (hot) {
        const char* row = a.logits + (int64_t)v.row * a.l_nb1 + (int64_t)s * a.l_nb2;
#pragma unroll
        for (int i = 0; i < kPer; i += Elem<TYPE>::per) load_vec<TYPE>(row, t0 + i, a.V, x + i);
    }
    const bool minus = v.d >= 0 && a.probs;
    if (minus) {
        const char* row = a.probs + (int64_t)v.row * a.p_nb1 + (int64_t)s * a.p_nb2;
        if (a.p_type == SIXI_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < kPer; i += 4) load_vec<SIXI_TYPE_F32>(row, t0 + i, a.V, q + i);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (t0 + i < a.V) q[i] = load1(row + (int64_t)(t0 + i) * 2, a.p_type);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int t = t0 + i;
        p[i] = hot ? weight(x[i], v.top, v.inv_t) * v.inv_z : v.inv_t == 0.0 && t == v.at ? 1.0 : 0.0;
        if (t >= a.V) p[i] = 0.0;
        w[i] = p[i];
        if (v.d >= 0) {
            const double less = minus ? p[i] - (double)q[i] : t == v.d ? p[i] - 1.0 : p[i];
            w[i] = less > 0.0 ? less : 0.0;
            if (t >= a.V) w[i] = 0.0;
        }
    }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void draft_draw_kernel(DraftArgs a) {
    __shared__ double ws[kThreads / 64], ps[kThreads / 64];
    __shared__ int lws[kThreads / 64], lps[kThreads / 64], stop;
    const int chunk = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
    const int rows = rows_of(a, s);
    if (rows == 0) {
        if (chunk == 0 && tid == 0) {
            a.keep[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    const DraftVerdict v = decide(a, s, rows, &stop);
    if (chunk == 0 && tid == 0) {
        a.keep[s] = v.row + 1;
        a.verdicts[s] = v;  // for the last launch
    }
    double w[kPer], p[kPer];
    const int t0 = chunk * kDraftChunk + tid * kPer;
    weights_of<TYPE>(a, s, v, t0, w, p);
    double sum_w = 0.0, sum_p = 0.0;
    int last_w = -1, last_p = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        sum_w += w[i];
        sum_p += p[i];
        if (w[i] > 0.0) last_w = t0 + i;
        if (p[i] > 0.0) last_p = t0 + i;
    }
    sum_w = wave_sum(sum_w);
    sum_p = wave_sum(sum_p);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        last_w = max(last_w, __shfl_xor(last_w, o, 64));
        last_p = max(last_p, __shfl_xor(last_p, o, 64));
    }
    if (tid % 64 == 0) {
        ws[tid / 64] = sum_w;
        ps[tid / 64] = sum_p;
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

// The sum of the lanes in front of one's own (a wave's running sum, by doubling steps).
__device__ __forceinline__ double wave_before(double x, double& total) {
    const int lane = threadIdx.x & 63;
    double run = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(run, o, 64);
        if (lane >= o) run += y;
    }
    total = __shfl(run, 63, 64);
    const double y = __shfl_up(run, 1, 64);
    return lane > 0 ? y : 0.0;
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void draft_find_kernel(DraftArgs a) {
    __shared__ double sums[kThreads / 64];
    __shared__ int first;
    const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    if (rows_of(a, s) == 0) return;
    const DraftVerdict v = a.verdicts[s];
    const DraftDraw* d = a.draws + (int64_t)s * a.chunks;
    // totals of the draw's weights and of p, then the first chunk whose end is past the mark; where the sums'
    // rounding (or u_next = 1) leaves none, the last one with a weight.  Every wave does this alike.
    double total = 0.0, total_p = 0.0;
    for (int c = lane; c < a.chunks; c += 64) {
        total += d[c].w;
        total_p += d[c].p;
    }
    total = wave_sum(total);
    total_p = wave_sum(total_p);
    const bool from_w = total > 0.0;
    if (!from_w) total = total_p;
    if (!(total > 0.0)) {
        if (tid == 0) a.token[s] = -1;
        return;
    }
    const double mark = (double)a.u_next[s] * total;
    double before = 0.0, ahead = 0.0;
    int chunk = 0, last = -1;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
        const int c = c0 + lane;
        const bool in = c < a.chunks;
        const double mine = in ? (from_w ? d[c].w : d[c].p) : 0.0;
        const int tail = in ? (from_w ? d[c].last_w : d[c].last_p) : -1;
        double sum;
        const double at = ahead + wave_before(mine, sum);
        const uint64_t some = __builtin_amdgcn_ballot_w64(tail >= 0), past = __builtin_amdgcn_ballot_w64(tail >= 0 && at + mine > mark);
        if (some) {
            const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
            chunk = c0 + l;
            before = __shfl(at, l, 64);
            last = __shfl(tail, l, 64);
        }
        if (past) break;
        ahead += sum;
    }
    // 16 consecutive tokens per thread, and the running sum over the threads
    const int t0 = chunk * kDraftChunk + tid * kPer;
    double w[kPer], p[kPer];
    weights_of<TYPE>(a, s, v, t0, w, p);
    double mine = 0.0, sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine += from_w ? w[i] : p[i];
    double at = wave_before(mine, sum);
    if (lane == 63) sums[tid / 64] = sum;
    if (tid == 0) first = kThreads;
    __syncthreads();
    double front = before;
    for (int k = 0; k < tid / 64; ++k) front += sums[k];
    at += front;
    if (mine > 0.0 && at + mine > mark) atomicMin(&first, tid);
    __syncthreads();
    if (first == kThreads) {  // (the chunk's end is past the mark by less than its sums' rounding)
        if (tid == 0) a.token[s] = last;
    } else if (tid == first) {
        int found = -1;
        bool done = false;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const double x = from_w ? w[i] : p[i];
            if (!done && x > 0.0) {
                at += x;
                found = t0 + i;
                done = at > mark;
            }
        }
        a.token[s] = found;
    }
}

template <int TYPE>
hipError_t launch(const DraftArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(draft_rows_kernel<TYPE>, dim3((unsigned)a.chunks, (unsigned)a.n_rows, (unsigned)a.S), dim3(kThreads), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(draft_draw_kernel<TYPE>, dim3((unsigned)a.chunks, (unsigned)a.S), dim3(kThreads), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(draft_find_kernel<TYPE>, dim3((unsigned)a.S), dim3(kThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_draft_verify(const DraftArgs& a, hipStream_t stream) {
    if (a.S == 0) return hipSuccess;
    if (a.l_type == SIXI_TYPE_F32) return launch<SIXI_TYPE_F32>(a, stream);
    if (a.l_type == SIXI_TYPE_F16) return launch<SIXI_TYPE_F16>(a, stream);
    return launch<SIXI_TYPE_BF16>(a, stream);
}

}  // namespace sixi
