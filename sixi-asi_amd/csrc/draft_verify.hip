// draft_verify.hip -- which drafted tokens stay, and the token behind them (include/sixi_draft.h).
//
// Two launches, a function of the inputs alone (every sum in a fixed order):
//   rows    every row's chunks of 4096 logits: largest, its token (where a greedy stream asks for it), sum of
//           2^((l - max) log2(e) / T)
//   draw    per stream, the accept chain from those sums (a few hundred numbers, formed again by each
//           work-group), then the chunk's share of the row that the next token is drawn from; the stream's
//           last work-group to get there finds the chunk and the token at which the running sum passes
//           u_next * total
// Bound by 64-bit arithmetic beside HBM (the logits once; the row that is drawn from a second time, out of the
// caches): 32 streams of 8 to 16 rows of 131072 f32 logits are 210 MB, 46 us for the rows (4.4 TB/s, the VALU busy
// for 70 % of them) and 24 for the draw, which is a chain of lookups: sums, weights, the last work-group, its
// chunk.  One stream of 5 rows: 4.5 and 12.5 us.  Sums and
// exponentials run in 64 bits: a token is found between neighbours of a running sum over the whole
// vocabulary, where 1e-7 of the total spans many of them.  2^x is its whole part, from the sum with 1.5 * 2^52,
// added to the exponent of a polynomial of degree 8 in the rest (Chebyshev interpolation on +-1/2: off by at
// most 1.1e-12): 14 f64 instructions, next to the loads.
#include <hip/hip_runtime.h>

#include "draft_internal.hpp"
#include "sixi_draft.h"

namespace sixi {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = kDraftChunk / kThreads;  // logits per thread
constexpr double kLog2e = 1.4426950408889634;

// The polynomial of 2^x on [-1/2, 1/2], highest power first.
constexpr double kPoly[9] = {1.3259565309065025e-06, 1.5310080791697267e-05, 0.00015403434142954517, 0.0013333450562298989, 0.009618129193338041,
                             0.055504109412126475, 0.2402265069564321, 0.6931471805459314, 1.0000000000000133};

// 2^y for y <= 0 (0 below -1000 and for NaN)
__device__ __forceinline__ double exp2_neg(double y) {
    constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are y's nearest whole number
    const double z = fmax(y, -1000.0), t = z + kWhole, r = z - (t - kWhole);
    double p = kPoly[0];
#pragma unroll
    for (int k = 1; k < 9; ++k) p = fma(p, r, kPoly[k]);
    p = __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
    return y > -1000.0 ? p : 0.0;
}

// exp((l - top) / T) with c = log2(e) / T; 0 for -inf and NaN.  Where the top is infinite, its equals take all.
__device__ __forceinline__ double weight(float l, float top, double c) {
    if (top == __builtin_huge_valf()) return l == top ? 1.0 : 0.0;
    return exp2_neg(((double)l - (double)top) * c);
}

__device__ __forceinline__ float load1(const char* p, int type) {
    if (type == SIXI_TYPE_F32) return *reinterpret_cast<const float*>(p);
    const uint16_t h = *reinterpret_cast<const uint16_t*>(p);
    if (type == SIXI_TYPE_F16) return (float)__builtin_bit_cast(_Float16, h);
    return __builtin_bit_cast(float, (uint32_t)h << 16);
}
__device__ __forceinline__ int bytes_of(int type) { return type == SIXI_TYPE_F32 ? 4 : 2; }

// A stream's temperature: 0 for a greedy one (NaN too), at most the largest finite number.
__device__ __forceinline__ float heat_of(const DraftArgs& a, int s) {
    const float t = a.temperature ? a.temperature[s] : 1.0f;
    return t > 0.0f ? fminf(t, 3.4028235e38f) : 0.0f;
}
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

// Moves within the 16 lanes of a row (DPP), and reductions and running sums from them: a few cycles a step,
// where a shuffle through LDS takes a hundred.
template <int CTRL>
__device__ __forceinline__ int dpp(int x, int none) {
    return __builtin_amdgcn_update_dpp(none, x, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x, float none) {
    return __int_as_float(dpp<CTRL>(__float_as_int(x), __float_as_int(none)));
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x, double none) {
    return __hiloint2double(dpp<CTRL>(__double2hiint(x), __double2hiint(none)), dpp<CTRL>(__double2loint(x), __double2loint(none)));
}
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140, kShr1 = 0x111;
__device__ __forceinline__ int lane_of(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ float lane_of(float x, int l) { return __int_as_float(lane_of(__float_as_int(x), l)); }
__device__ __forceinline__ double lane_of(double x, int l) { return __hiloint2double(lane_of(__double2hiint(x), l), lane_of(__double2loint(x), l)); }

// f over the 16 lanes of a row, then over the wave's four rows; the result in every lane.
template <typename T, typename F>
__device__ __forceinline__ T row_reduce(T x, F f) {
    x = f(x, dpp<kXor1>(x, x));
    x = f(x, dpp<kXor2>(x, x));
    x = f(x, dpp<kHalfMirror>(x, x));
    return f(x, dpp<kMirror>(x, x));
}
template <typename T, typename F>
__device__ __forceinline__ T wave_reduce(T x, F f) {
    x = row_reduce(x, f);
    return f(f(lane_of(x, 0), lane_of(x, 16)), f(lane_of(x, 32), lane_of(x, 48)));
}
struct Plus {
    __device__ __forceinline__ double operator()(double a, double b) const { return a + b; }
};
struct Greater {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
    __device__ __forceinline__ int operator()(int a, int b) const { return max(a, b); }
};
struct Less {
    __device__ __forceinline__ int operator()(int a, int b) const { return min(a, b); }
};

// The sum of the lanes in front of one's own, and of all.
__device__ __forceinline__ double wave_before(double x, double& total) {
    double run = x;
    run += dpp<0x111>(run, 0.0);
    run += dpp<0x112>(run, 0.0);
    run += dpp<0x114>(run, 0.0);
    run += dpp<0x118>(run, 0.0);
    const double r0 = lane_of(run, 15), r1 = lane_of(run, 31), r2 = lane_of(run, 47), r3 = lane_of(run, 63);
    const int row = (threadIdx.x & 63) >> 4;
    const double front = row == 0 ? 0.0 : row == 1 ? r0 : row == 2 ? r0 + r1 : (r0 + r1) + r2;
    total = ((r0 + r1) + r2) + r3;
    return dpp<kShr1>(run, 0.0) + front;
}

// exp2_neg's sum over a thread's logits, for a total only: what is hidden or far below counts 2^-1000.
__device__ __forceinline__ double sum_of(const float (&x)[kPer], float top, double c, float least) {
    constexpr double kWhole = 6755399441055744.0;
    const double off = -(double)top * c;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const double y = fma((double)fmaxf(x[i], least), c, off), t = y + kWhole, r = y - (t - kWhole);
        double p = kPoly[0];
#pragma unroll
        for (int k = 1; k < 9; ++k) p = fma(p, r, kPoly[k]);
        sum += __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
    }
    return sum;
}

// A work-group takes a.run chunks of a row, the next one's loads ahead of the sums over the last; its waves go
// by themselves, each with a running maximum and a sum relative to it, and are joined behind the only barrier.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void draft_rows_kernel(DraftArgs a) {
    constexpr int kVec = Elem<TYPE>::per, kWaves = kThreads / 64;
    __shared__ float tops[kWaves];
    __shared__ int ats[kWaves];
    __shared__ double sums[kWaves];
    const int part = blockIdx.x, j = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    if (j >= rows_of(a, s)) return;
    if (part == 0 && j == 0 && tid == 0) a.counts[s] = 0;  // for the next launch
    const char* row = a.logits + (int64_t)j * a.l_nb1 + (int64_t)s * a.l_nb2;
    const float heat = heat_of(a, s);
    const bool hot = heat > 0.0f;
    const double c = hot ? kLog2e / (double)heat : 0.0;
    const float span = hot ? (float)(1000.0 / c) : 0.0f;
    const int first = part * a.run, last = min(first + a.run, a.chunks);
    const float none = -__builtin_huge_valf();
    float top = none;
    int at = a.V;
    double sum = 0.0;
    float next[kPer];
    auto load = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < kPer; i += kVec) load_vec<TYPE>(row, chunk * kDraftChunk + i * kThreads + tid * kVec, a.V, next + i);
    };
    load(first);
    for (int chunk = first; chunk < last; ++chunk) {
        float x[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) x[i] = next[i];
        if (chunk + 1 < last) load(chunk + 1);
        float here = x[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i) here = fmaxf(here, x[i]);  // (fmaxf passes over NaN)
        here = wave_reduce(here, Greater());
        if (!(here > none)) continue;  // (nothing but -inf and NaN)
        if (!hot) {
            if (here > top) {
                int h = a.V;
#pragma unroll
                for (int i = kPer - 1; i >= 0; --i)
                    if (x[i] == here) h = min(h, chunk * kDraftChunk + i / kVec * kVec * kThreads + tid * kVec + i % kVec);
                at = wave_reduce(h, Less());
                top = here;
            }
        } else if (here == __builtin_huge_valf()) {  // infinite logits share everything
            double n = 0.0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) n += x[i] == here ? 1.0 : 0.0;
            sum = top == here ? sum + n : n;
            top = here;
        } else if (top < __builtin_huge_valf()) {
            if (here > top) {
                sum *= weight(top, here, c);
                top = here;
            }
            // (temperatures whose 1000 powers of two are a few steps of the top, or past the type: one by one)
            if (span >= fabsf(top) * 0x1p-18f && span < 1e30f && fabsf(top) < 1e30f) {
                sum += sum_of(x, top, c, top - span);
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i) sum += weight(x[i], top, c);
            }
        }
    }
    sum = wave_reduce(sum, Plus());
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
        if (hot && best > none) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) z += sums[w] * weight(tops[w], best, c);
        }
        DraftPart& p = a.parts[((int64_t)s * a.n_rows + j) * a.n_parts + part];
        p.sum = z;
        p.top = best;
        p.at = best_at;
    }
}

constexpr int kGroup = 16;  // lanes that sum a row's chunks

struct RowSum {
    double z;
    float top;
    int at;
    int d;  // the row's drafted token, -1 for none
};
// A row's largest logit and sum of weights, by the 16 lanes of a group (every lane gets them).
__device__ __forceinline__ RowSum row_sum(const DraftArgs& a, int s, int j, double c) {
    const int lane = threadIdx.x % kGroup;
    const DraftPart* parts = a.parts + ((int64_t)s * a.n_rows + j) * a.n_parts;
    RowSum r{0.0, -__builtin_huge_valf(), a.V, -1};
#pragma unroll 4
    for (int i = lane; i < a.n_parts; i += kGroup) take_top(r.top, r.at, parts[i].top, parts[i].at);
    const float mine = r.top;
    r.top = row_reduce(mine, Greater());
    r.at = row_reduce(mine == r.top ? r.at : a.V, Less());
#pragma unroll 2
    for (int i = lane; i < a.n_parts; i += kGroup) r.z += parts[i].sum * weight(parts[i].top, r.top, c);
    r.z = row_reduce(r.z, Plus());
    return r;
}

// Each group of 16 lanes judges rows of its own; `stop` is then the first whose token goes, or the last
// row.  Every thread of the work-group calls this; `sums` (a row each) and `stop` are in LDS.
__device__ __forceinline__ DraftVerdict decide(const DraftArgs& a, int s, int rows, RowSum* sums, int* stop) {
    const float heat = heat_of(a, s);
    DraftVerdict v{};
    v.c = heat > 0.0f ? kLog2e / (double)heat : 0.0;
    if (threadIdx.x == 0) *stop = rows - 1;
    __syncthreads();
    for (int j = threadIdx.x / kGroup; j < rows; j += kThreads / kGroup) {
        float l = 0.0f, u = 0.0f;
        double p = 0.0, q = 1.0;
        int d = -1;
        if (j < rows - 1) {
            d = a.draft[(int64_t)s * a.draft_stride + j];
            u = a.u[(int64_t)s * a.u_stride + j];
        }
        const bool known = d >= 0 && d < a.V;
        if (known) {
            l = load1(a.logits + (int64_t)j * a.l_nb1 + (int64_t)s * a.l_nb2 + (int64_t)d * bytes_of(a.l_type), a.l_type);
            if (a.probs)
                q = load1(a.probs + (int64_t)j * a.p_nb1 + (int64_t)s * a.p_nb2 + (int64_t)d * bytes_of(a.p_type), a.p_type);
        }
        RowSum r = row_sum(a, s, j, v.c);
        r.d = d;
        if (threadIdx.x % kGroup == 0) {
            sums[j] = r;
            if (known) p = v.c == 0.0 ? (d == r.at ? 1.0 : 0.0) : r.z > 0.0 ? weight(l, r.top, v.c) / r.z : 0.0;
            if (j < rows - 1 && !((double)u * q < p)) atomicMin(stop, j);
        }
    }
    __syncthreads();
    // (the same in all lanes, and known to be: scalar registers and branches from here on)
    v.row = lane_of(*stop, 0);
    const RowSum r = sums[v.row];
    const int d = lane_of(r.d, 0);
    const double z = lane_of(r.z, 0);
    v.top = lane_of(r.top, 0);
    v.at = lane_of(r.at, 0);
    v.inv_z = z > 0.0 ? 1.0 / z : 0.0;
    v.d = -1;
    if (v.row < rows - 1) v.d = d >= 0 && d < a.V ? d : a.V;
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
    const bool hot = v.c != 0.0 && v.top > -__builtin_huge_valf();
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
        } else if (a.p_type == SIXI_TYPE_F16) {
#pragma unroll
            for (int i = 0; i < kPer; i += 8) load_vec<SIXI_TYPE_F16>(row, t0 + i, a.V, q + i);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; i += 8) load_vec<SIXI_TYPE_BF16>(row, t0 + i, a.V, q + i);
        }
    }
    // (no branch between the tokens: their polynomials run next to one another)
    const bool all = v.top == __builtin_huge_valf();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        double y = ((double)x[i] - (double)v.top) * v.c;
        if (all) y = x[i] == v.top ? 0.0 : -2000.0;
        p[i] = exp2_neg(y) * v.inv_z;  // (0 past the end: -inf there)
    }
    if (!hot) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) p[i] = v.c == 0.0 && t0 + i == v.at ? 1.0 : 0.0;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const double less = minus ? p[i] - (double)fmaxf(q[i], 0.0f) :  // (-inf past the end)
                                     t0 + i == v.d ? p[i] - 1.0 : p[i];
        w[i] = v.d < 0 ? p[i] : fmax(less, 0.0);
    }
}

// What other work-groups wrote in the same launch: loads and stores at the device's scope, past the caches
// that are not shared.
__device__ __forceinline__ void put(DraftDraw* d, const DraftDraw& x) {
    __hip_atomic_store(&d->w, x.w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&d->p, x.p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&d->last_w, x.last_w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&d->last_p, x.last_p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ DraftDraw get(DraftDraw* d) {
    return {__hip_atomic_load(&d->w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT), __hip_atomic_load(&d->p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
            __hip_atomic_load(&d->last_w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT),
            __hip_atomic_load(&d->last_p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)};
}

// Where the running sum passes the mark: the chunk, the sum in front of it, its last token with a weight.
struct DraftFound {
    double mark, before;
    int chunk, last;  // chunk -1: no weight at all
    bool from_w;
};
// The first chunk whose end is past the mark; where the sums' rounding (or u_next = 1) leaves none, the last one
// with a weight.  Every wave does this alike.
__device__ __forceinline__ DraftFound find_chunk(const DraftArgs& a, int s, double u_next) {
    const int lane = threadIdx.x & 63;
    DraftDraw* draws = a.draws + (int64_t)s * a.chunks;
    const DraftDraw none{0.0, 0.0, -1, -1};
    const DraftDraw mine0 = lane < a.chunks ? get(draws + lane) : none;  // (most vocabularies: all there is)
    double total = mine0.w, total_p = mine0.p;
    for (int c = lane + 64; c < a.chunks; c += 64) {
        const DraftDraw d = get(draws + c);
        total += d.w;
        total_p += d.p;
    }
    total = wave_reduce(total, Plus());
    total_p = wave_reduce(total_p, Plus());
    DraftFound f{0.0, 0.0, -1, -1, total > 0.0};
    if (!f.from_w) total = total_p;
    if (!(total > 0.0)) return f;
    f.mark = u_next * total;
    double ahead = 0.0;
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
        const DraftDraw d = c0 == 0 ? mine0 : c0 + lane < a.chunks ? get(draws + c0 + lane) : none;
        const double mine = f.from_w ? d.w : d.p;
        const int tail = f.from_w ? d.last_w : d.last_p;
        double sum;
        const double at = ahead + wave_before(mine, sum);
        const uint64_t some = __builtin_amdgcn_ballot_w64(tail >= 0), past = __builtin_amdgcn_ballot_w64(tail >= 0 && at + mine > f.mark);
        if (some) {
            const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
            f.chunk = c0 + l;
            f.before = lane_of(at, l);
            f.last = lane_of(tail, l);
        }
        if (past) break;
        ahead += sum;
    }
    return f;
}

// A stream's chunks, a.draw_run to a work-group; the last work-group goes through the chunk found once more.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void draft_draw_kernel(DraftArgs a) {
    __shared__ double ws[kThreads / 64], ps[kThreads / 64];
    __shared__ int lws[kThreads / 64], lps[kThreads / 64], stop, last;
    __shared__ RowSum sums[kDraftMaxRows];
    const int s = blockIdx.y, tid = threadIdx.x;
    const int rows = rows_of(a, s);
    if (rows == 0) {
        if (blockIdx.x == 0 && tid == 0) {
            a.keep[s] = 0;
            a.token[s] = -1;
        }
        return;
    }
    const double u_next = (double)a.u_next[s];
    const DraftVerdict v = decide(a, s, rows, sums, &stop);
    if (blockIdx.x == 0 && tid == 0) a.keep[s] = v.row + 1;
    const int first = blockIdx.x * a.draw_run, end = min(first + a.draw_run, a.chunks);
    DraftFound f{0.0, 0.0, first, -1, true};
    bool found = false;
#pragma unroll 1
    while (true) {
        // 16 consecutive tokens per thread
        double w[kPer], p[kPer];
        const int t0 = f.chunk * kDraftChunk + tid * kPer;
        weights_of<TYPE>(a, s, v, t0, w, p);
        if (!found) {
            double sum_w = 0.0, sum_p = 0.0;
            int last_w = -1, last_p = -1;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                sum_w += w[i];
                sum_p += p[i];
                if (w[i] > 0.0) last_w = t0 + i;
                if (p[i] > 0.0) last_p = t0 + i;
            }
            sum_w = wave_reduce(sum_w, Plus());
            sum_p = wave_reduce(sum_p, Plus());
            last_w = wave_reduce(last_w, Greater());
            last_p = wave_reduce(last_p, Greater());
            if (tid % 64 == 0) {
                ws[tid / 64] = sum_w;
                ps[tid / 64] = sum_p;
                lws[tid / 64] = last_w;
                lps[tid / 64] = last_p;
            }
            __syncthreads();
            if (tid == 0) {
                put(a.draws + (int64_t)s * a.chunks + f.chunk,
                    {((ws[0] + ws[1]) + ws[2]) + ws[3], ((ps[0] + ps[1]) + ps[2]) + ps[3], max(max(lws[0], lws[1]), max(lws[2], lws[3])),
                     max(max(lps[0], lps[1]), max(lps[2], lps[3]))});
                if (f.chunk + 1 == end) {
                    // counted once the stores above have reached the device's memory
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    last = __hip_atomic_fetch_add(a.counts + s, end - first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + end - first == a.chunks;
                }
            }
            __syncthreads();
            if (++f.chunk < end) continue;
            if (!last) return;
            found = true;
            f = find_chunk(a, s, u_next);
            if (f.chunk < 0) {
                if (tid == 0) a.token[s] = -1;
                return;
            }
            continue;
        }
        // the running sum over the threads, then over the tokens of the thread that passes the mark
        double mine = 0.0, sum;
#pragma unroll
        for (int i = 0; i < kPer; ++i) mine += f.from_w ? w[i] : p[i];
        double at = wave_before(mine, sum);
        if (tid % 64 == 63) ws[tid / 64] = sum;
        if (tid == 0) stop = kThreads;
        __syncthreads();
        double front = f.before;
        for (int k = 0; k < tid / 64; ++k) front += ws[k];
        at += front;
        if (mine > 0.0 && at + mine > f.mark) atomicMin(&stop, tid);
        __syncthreads();
        if (stop == kThreads) {  // (the chunk's end is past the mark by less than its sums' rounding)
            if (tid == 0) a.token[s] = f.last;
        } else if (tid == stop) {
            int token = -1;
            bool done = false;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const double x = f.from_w ? w[i] : p[i];
                if (!done && x > 0.0) {
                    at += x;
                    token = t0 + i;
                    done = at > f.mark;
                }
            }
            a.token[s] = token;
        }
        return;
    }
}

template <int TYPE>
hipError_t launch(const DraftArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(draft_rows_kernel<TYPE>, dim3((unsigned)a.n_parts, (unsigned)a.n_rows, (unsigned)a.S), dim3(kThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(draft_draw_kernel<TYPE>, dim3((unsigned)((a.chunks + a.draw_run - 1) / a.draw_run), (unsigned)a.S), dim3(kThreads), 0, stream, a);
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
