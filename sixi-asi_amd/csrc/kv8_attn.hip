// kv8_attn.hip -- attention over the 8-bit cache (include/sixi_kv8.h).
//
// One pass over the cells with the running maximum and sum of a softmax.  A group's rows (row j of the
// G heads that share a kv-head; row index r = j * G + h) are taken 32 at a time as the columns of
//   S^T[cell, row] = K Q^T      O^T[dim, row] += V^T P^T
// on v_mfma_f32_32x32x16_f16, a block of 32 cells per step.  Both left operands come from the cache as
// it lies in memory: 16 bytes per lane, 1 KiB per wave.  Codes become f16 exactly (|code| <= 127), the
// scales are powers of two and never meet an element:
//   t = scale log2(e) 2^ek (q . k) + ev        the exponent of (weight * 2^ev)
//   P' = 2^(t - m)                              m a reference near the running maximum of t
//   O' = sum P' v,   l = sum P' 2^-ev,   o = O' / l
// With ev inside the exponent a block's V scale costs nothing, and the f16 rounding of P' is half a step
// of 11 bits of each weight, down to 2^-24 of the largest contribution whatever the blocks' scales are.
// l is the f32 sum of the weights in front of that rounding: a block with a small V scale stands next to
// one with a large one, and its f16 weights would be too coarse for the sum they are most of.
//
// The cell that score register i of a lane holds is ours to choose (any order of K's rows will do):
// lane (n, h) of the 32 x 32 result holds cells 16h .. 16h + 15 of the block in order, which is what the
// lane needs as its half of the next product's right operand.  So P never leaves its lane.
//
// Two forms.  Up to 32 rows a group (decode), or 64 of 128 dims: the four waves of a work-group take blocks
// in turn, straight from memory into registers, one block ahead; nothing is shared but the queries.
// More rows: four waves take 32 rows each of the same cells; a step's codes are converted once, by all of them,
// into f16 operands in LDS, the next step's codes on their way in registers (a kernel for each head dim).
//
// Work-groups: every stream's cells are cut into pieces of c blocks, c from the lengths on the device, so
// that streams of any lengths fill the chip; pieces of one (stream, head, tile) are joined by a second
// launch in their order.
#include <algorithm>
#include <type_traits>

#include "device_util.hpp"
#include "kv8_device.hpp"

namespace sixi {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3e38f;  // below every score: the reference of a row that has seen no cell
// The largest weight stands between 2^kHead and 2^kRoof: f16 weights keep 11 bits down to 2^-24 of 2^kHead,
// and the accumulators are rescaled only when a maximum has grown by 2^(kRoof - kHead).
constexpr float kHead = 10.0f, kRoof = 15.0f;

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
__device__ __forceinline__ int blocks_of(const Lens& n) { return (n.cells + kBlk - 1) / kBlk; }

// Whether tiles are nearly a work-group for every place there is: then no cells are cut.
__device__ __host__ __forceinline__ bool enough(int64_t tiles, const Kv8AttnArgs& a) {
    return 4 * tiles * a.Hkv >= 3 * (int64_t)a.target;
}

// How a call's cells are cut: pieces of c blocks, numbered stream by stream.  c is the work of
// all streams over the work-groups asked for; nothing is cut where the tiles alone are nearly enough of
// them.  Whole numbers, formed alike by every work-group of a call.
typedef Kv8Place Place;
struct Cut {
    int c, total;
    // of the lane's stream (S <= 64), else of the last 64 looked at
    int tiles, pieces, at, mine;

    __device__ __forceinline__ void stream(const Kv8AttnArgs& a, int s, int& t, int& blocks) const {
        t = blocks = 0;
        if (s < a.S) {
            const Lens n = lens_of(a, s);
            t = (n.rows * a.G + 32 * a.waves - 1) / (32 * a.waves);
            blocks = blocks_of(n);
        }
    }
    __device__ __forceinline__ void count(const Kv8AttnArgs& a, int t, int blocks, int before) {
        tiles = t;
        pieces = max(1, (blocks + c - 1) / c);
        mine = t * pieces * a.Hkv;
        const int run = wave_scan(mine);
        at = before + run - mine;
        total = before + __builtin_amdgcn_readlane(run, 63);
    }
    __device__ __forceinline__ void begin(const Kv8AttnArgs& a) {
        const int lane = threadIdx.x & 63;
        int t = 0, blocks = 0, all = 0, work = 0;
        // a stream's share of a work-group's blocks, in 1/64 (f32, and then whole numbers: the same sum in
        // every work-group; where cells are cut it is at most 0.75 * 64 * 2^21 blocks in all)
        const float unit = 64.0f * (float)a.Hkv / (float)a.target;
        for (int s0 = 0; s0 < a.S; s0 += 64) {
            stream(a, s0 + lane, t, blocks);
            all += __builtin_amdgcn_readlane(wave_scan(t), 63);
            work += __builtin_amdgcn_readlane(wave_scan((int)fminf((float)t * (float)blocks * unit, 134217728.0f) + 1), 63);
        }
        // even: two blocks a step, and of one page
        c = enough(all, a) ? 1 << 26 : (max((work + 63) / 64, a.least) + 1) / 2 * 2;
        // every stream's last piece is a part of one: longer pieces until they fit the places there are
        for (int tries = 0;; ++tries) {
            total = 0;
            if (a.S <= 64)
                count(a, t, blocks, 0);
            else
                for (int s0 = 0; s0 < a.S; s0 += 64) {
                    stream(a, s0 + lane, t, blocks);
                    count(a, t, blocks, total);
                }
            if (total <= a.target || c >= 1 << 26 || tries == 3) return;
            c = (int)((float)c * fminf((float)total / (float)a.target, 1.5f)) / 2 * 2 + 2;
        }
    }
    // The same for a call of one stream.
    __device__ __forceinline__ void alone(const Kv8AttnArgs& a, Place& p) {
        const Lens n = lens_of(a, 0);
        const int t = (n.rows * a.G + 32 * a.waves - 1) / (32 * a.waves), blocks = blocks_of(n), all = t * a.Hkv;
        // as many pieces as fit the places beside the other tiles and heads
        const int most = enough(t, a) ? 1 : a.target / max(all, 1);
        c = (max((blocks + most - 1) / most, a.least) + 1) / 2 * 2;
        p.tiles = t;
        p.pieces = max(1, (blocks + c - 1) / c);
        total = all * p.pieces;
    }
    // The stream that holds piece `id`.
    __device__ __forceinline__ Place find(const Kv8AttnArgs& a, int id) {
        const int lane = threadIdx.x & 63, sum = total;
        Place p{0, 1, 1, 0};
        int before = 0;
        for (int s0 = 0; s0 < a.S; s0 += 64) {
            if (a.S > 64) {
                int t, blocks;
                stream(a, s0 + lane, t, blocks);
                count(a, t, blocks, before);
                before = total;
            }
            const uint64_t hit = __builtin_amdgcn_ballot_w64(id >= at && id < at + mine);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                p.s = s0 + l;
                p.tiles = __builtin_amdgcn_readlane(tiles, l);
                p.pieces = __builtin_amdgcn_readlane(pieces, l);
                p.at = __builtin_amdgcn_readlane(at, l);
                break;
            }
        }
        total = sum;
        return p;
    }
};

// Floats of a piece's partial result: per wave-tile of 32 rows, O in the order of the accumulators
// [D/8][64 lanes][4], then m and l of 32 rows.
__device__ __host__ constexpr int64_t tile_floats(int D) { return 32 * (int64_t)D + 64; }

__device__ __forceinline__ void store4(const Kv8AttnArgs& a, char* row, int d, kv8_f32x4 x) {
    if (a.o_f16) {
        f16x4 h;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = (_Float16)x[i];
        *reinterpret_cast<f16x4*>(row + d * 2) = h;
    } else {
        *reinterpret_cast<kv8_f32x4*>(row + d * 4) = x;
    }
}

// Which row of a group's 32 is the lane's: row j of the block, q-head `head`.
struct Seat {
    int j, head;
    bool live;
};
__device__ __forceinline__ Seat seat_of(const Kv8AttnArgs& a, const Lens& n, int g, int r0) {
    const int r = r0 + (threadIdx.x & 31);
    const bool live = r < n.rows * a.G;
    return {live ? r / a.G : 0, g * a.G + (live ? r % a.G : 0), live};
}

// What a wave holds of 32 rows of a group: their sums.
template <int D>
struct Rows {
    static constexpr int KC = D / 32;  // 32-dim pieces of a row: K loads, V loads and output tiles
    f32x16 o[KC];
    float m, l;
    int last;     // the last cell that the lane's row sees
    int sees;     // the last cell that every row sees
    int reach;    // cells that any of the rows sees

    __device__ __forceinline__ void begin(const Kv8AttnArgs& a, const Lens& n, int r0, const Seat& x) {
        const int M = n.rows * a.G;
        const bool causal = a.mode == SIXI_MASK_BLOCK_CAUSAL;
        last = causal ? n.cached + x.j : n.cells - 1;
        sees = causal ? n.cached + r0 / a.G : n.cells - 1;
        reach = causal ? n.cached + (min(r0 + 32, M) - 1) / a.G + 1 : n.cells;
        if (r0 >= M) reach = 0;
#pragma unroll
        for (int c = 0; c < KC; ++c) o[c] = f32x16{};
        m = kLowest;
        l = 0.0f;
    }

    // The rows' queries, 32 dims of them, as a product's right operands.
    __device__ __forceinline__ static void queries(const Kv8AttnArgs& a, int s, const Seat& seat, int c, kv8_f16x8 (&q)[2]) {
        const int h = (threadIdx.x & 63) >> 5;
        const char* p = a.q + (int64_t)seat.j * a.q_nb1 + (int64_t)seat.head * a.q_nb2 + (int64_t)s * a.q_nb3;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int d = (2 * c + h) * 16 + 8 * u;
            kv8_f16x8 x = {};
            if (seat.live) {
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
                x = x * (_Float16)a.q_sign;
            }
            q[u] = x;
        }
    }

    // The mask's values for the lane's 16 cells of a block (all of a block's are there, whatever the row sees).
    __device__ __forceinline__ static void mask_of(const char* mask, int block, f16x8u (&add)[2]) {
        const char* p = mask + (int64_t)(block * kBlk + 16 * ((threadIdx.x & 63) >> 5)) * 2;
        add[0] = *reinterpret_cast<const f16x8u*>(p);
        add[1] = *reinterpret_cast<const f16x8u*>(p + 16);
    }
    // A block's scores: hidden cells to -inf; with a mask, to t itself.
    template <bool MASK>
    __device__ __forceinline__ void hide(f32x16& sc, int block, float ks, float es, const f16x8u (&add)[2]) const {
        const int cell0 = block * kBlk + 16 * ((threadIdx.x & 63) >> 5);
        if (MASK) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] = fmaf(sc[i], ks, fmaf((float)add[i / 8][i % 8], kLog2e, es));
        }
        if (block * kBlk + kBlk - 1 > sees) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (cell0 + i > last) sc[i] = -__builtin_huge_valf();
        }
    }
    // The row's largest t of a block (maxima that keep NaN: no operand is canonicalised first).
    template <bool MASK>
    __device__ __forceinline__ float top_of(const f32x16& sc, float ks, float es) const {
        float top = __builtin_elementwise_maximum(sc[0], sc[1]), top2 = __builtin_elementwise_maximum(sc[2], sc[3]);
#pragma unroll
        for (int i = 4; i < 16; i += 4) {
            top = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top, sc[i]), sc[i + 1]);
            top2 = __builtin_elementwise_maximum(__builtin_elementwise_maximum(top2, sc[i + 2]), sc[i + 3]);
        }
        top = max_halves(__builtin_elementwise_maximum(top, top2));
        return MASK ? top : fmaf(top, ks, es);
    }
    // Scores to weights in f16, and their sum.
    template <bool MASK>
    __device__ __forceinline__ void weights(const f32x16& sc, float ks, float es, int ev, kv8_f16x8 (&p)[2]) {
        const float sub = MASK ? -m : es - m;
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            f32x2 w;
#pragma unroll
            for (int e = 0; e < 2; ++e) w[e] = __builtin_amdgcn_exp2f(MASK ? sc[i + e] + sub : fmaf(sc[i + e], ks, sub));
            const f16x2 x = __builtin_convertvector(w, f16x2);
            p[i / 8][i % 8] = x[0];
            p[i / 8][i % 8 + 1] = x[1];
            sum[0] += w[0];
            sum[1] += w[1];
        }
        l = fmaf(sum[0] + sum[1], exp2_int(-ev), l);
    }

    __device__ __forceinline__ void finish(const Kv8AttnArgs& a, int s, const Seat& seat) const {
        if (!seat.live) return;
        const int h = (threadIdx.x & 63) >> 5;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        char* row = a.out + (int64_t)seat.head * a.o_nb1 + (int64_t)seat.j * a.o_nb2 + (int64_t)s * a.o_nb3;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                store4(a, row, c * 32 + 2 * i + 4 * h, kv8_f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]} * inv);
    }

    __device__ __forceinline__ void leave(float* part, const Seat& seat) const {
        const int lane = threadIdx.x & 63;
        if (!seat.live) return;
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<kv8_f32x4*>(part + ((c * 4 + i / 4) * 64 + lane) * 4) =
                    kv8_f32x4{o[c][i], o[c][i + 1], o[c][i + 2], o[c][i + 3]};
        if (lane < 32) {
            part[32 * D + lane] = m;
            part[32 * D + 32 + lane] = l;
        }
    }
};

// A new reference where a maximum has outgrown the old one (a NaN has not; its weights are NaN).
template <int D, int T>
__device__ __forceinline__ void raise(Rows<D> (&r)[T], const float (&top)[T]) {
    bool grow = false;
#pragma unroll
    for (int t = 0; t < T; ++t) grow |= top[t] > r[t].m + kRoof;
    if (!__builtin_amdgcn_ballot_w64(grow)) return;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const float up = top[t] > r[t].m + kRoof ? top[t] - kHead : r[t].m, f = __builtin_amdgcn_exp2f(r[t].m - up);
        r[t].m = up;
        r[t].l *= f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) r[t].o[c] *= f;
    }
}

// The piece of a work-group, in the order (stream, tile from the last on, piece, head): the longest tiles of a
// causal chunk first, and, as work-groups go round the 8 XCDs, tiles of the same head on few of them, where
// they meet in the L2.
struct Work {
    int s, g, tile, id, first, last, pieces;
    Lens n;
};
__device__ __forceinline__ bool work_of(const Kv8AttnArgs& a, Work& w) {
    w.id = blockIdx.x;
    Cut cut;
    Place p{0, 1, 1, 0};
    if (a.S == 1) {  // one stream needs no sums over streams (0.4 us of a token behind 4095 cells)
        cut.alone(a, p);
        if (w.id >= cut.total) return false;
    } else {
        cut.begin(a);
        if (w.id >= cut.total) return false;
        p = cut.find(a, w.id);
    }
    if (a.cut && w.id == p.at && threadIdx.x == 0) a.places[p.s] = p;  // for the merge
    w.s = p.s;
    w.pieces = p.pieces;
    const int x = w.id - p.at;
    w.g = x % a.Hkv;
    const int y = x / a.Hkv, piece = y % p.pieces;
    w.tile = p.tiles - 1 - y / p.pieces;
    w.n = lens_of(a, w.s);
    w.first = piece * cut.c;
    w.last = min(blocks_of(w.n), w.first + cut.c);
    return true;
}

constexpr int kWaves = 4;

// 16 bytes of codes; ONCE: not to be kept in the caches.
template <bool ONCE>
__device__ __forceinline__ kv8_u32x4 codes_at(const char* p) {
    const kv8_u32x4* x = reinterpret_cast<const kv8_u32x4*>(p);
    return ONCE ? __builtin_nontemporal_load(x) : *x;
}

// T tiles of 32 rows in the registers of every wave, the waves on cells of their own; joined through LDS at the end.
// The queries are read from LDS in every step and K is converted piece by piece beside its products: with the
// accumulators that leaves room for two work-groups on a CU at 256 dims too, i.e. twice the codes on their way
// (32 streams behind 0.5k to 8k cells, 256 dims: 66 us, and 72 with the queries in registers and one; now 59).
//
// Bound by memory where streams are many or long: one token of 32 streams behind 0.5k to 16k cells, 128 dims, 269 MB:
// 53 us with the cut, the merge and its launch, 5.0 TB/s.  Bound by latency where they are not: one token
// behind 4095 cells, 256 dims: 14.2 us with the merge, of it lengths and cut 1.3, codes and queries 2.8, the step 2,
// the four waves' join 2.
// Two tiles, and loads that leave nothing in the caches (ONCE), are rules of kv8_attn_plan.
template <int D, int T, bool MASK, bool ONCE>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attn_few_kernel(Kv8AttnArgs a) {
    constexpr int KC = D / 32;
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!work_of(a, w)) return;
    // cells that any row sees
    int last = w.last;
    const int r0 = w.tile * (32 * T);
    if (a.mode == SIXI_MASK_BLOCK_CAUSAL)
        last = min(last, (w.n.cached + (min(r0 + 32 * T, w.n.rows * a.G) - 1) / a.G + kBlk) / kBlk);
    const uint32_t k_off = h * (kBlk * 16) + (16 * (n / 4 % 2) + 4 * (n / 8) + n % 4) * 16;
    const uint32_t v_off = n * kBlk + h * 16;

    // the first block's codes are asked for before the queries; from then on K of the next block when this
    // one's is f16, V when this one's is spent
    int b = w.first + wave;
    kv8_u32x4 kc[KC], vc[KC];
    int ek = 0, ev = 0;
    BlockWalk walk;
    if (b < last) {
        walk.begin(a.pages, a.k, a.v, w.s, w.g, b, last);
#pragma unroll
        for (int c = 0; c < KC; ++c) kc[c] = codes_at<ONCE>(walk.k + k_off + c * (kBlk * 32));
        ek = *walk.ke;
        ev = *walk.ve;
#pragma unroll
        for (int c = 0; c < KC; ++c) vc[c] = codes_at<ONCE>(walk.v + v_off + c * (kBlk * 32));
    }
    Rows<D> r[T];
    Seat seat[T];
    const char* mask[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        seat[t] = seat_of(a, w.n, w.g, r0 + t * 32);
        r[t].begin(a, w.n, r0 + t * 32, seat[t]);
        mask[t] = MASK ? a.mask + (int64_t)seat[t].j * a.m_nb1 + (int64_t)w.s * a.m_nb3 : nullptr;
    }
    // the queries stay in LDS, for all waves, each of which fetches a share: [tile][piece][first, second eight][lane]
    typedef kv8_f16x8 Queries[KC][2][64];
    Queries* qs = reinterpret_cast<Queries*>(lds);
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int c = 0; c < KC; c += kWaves) {
            kv8_f16x8 q[2];
            Rows<D>::queries(a, w.s, seat[t], c + wave, q);
            qs[t][c + wave][0][lane] = q[0];
            qs[t][c + wave][1][lane] = q[1];
        }
    __syncthreads();
    if (b < last) {
        f16x8u add[T][2], next[T][2];
        if (MASK)
#pragma unroll
            for (int t = 0; t < T; ++t) Rows<D>::mask_of(mask[t], b, next[t]);
        walk.go(a.pages, a.k, a.v, w.s, w.g, kWaves);
        for (; b < last; b += kWaves) {
            f32x16 sc[T] = {};
            int at = lane;  // (read from LDS in every step: out of the loop they would fill the registers)
            asm volatile("" : "+v"(at));
            const int ek0 = clamp_exp(ek), ev0 = clamp_exp(ev);
            ek = *walk.ke;
            ev = *walk.ve;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                kv8_f16x8 x[2];
                codes_f16x16(kc[c], x[0], x[1]);
                kc[c] = codes_at<ONCE>(walk.k + k_off + c * (kBlk * 32));
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int t = 0; t < T; ++t) sc[t] = mfma(x[u], qs[t][c][u][at], sc[t]);
            }
            if (MASK)
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    add[t][0] = next[t][0];
                    add[t][1] = next[t][1];
                    Rows<D>::mask_of(mask[t], walk.b, next[t]);
                }
            const char* vn = walk.v;
            walk.go(a.pages, a.k, a.v, w.s, w.g, kWaves);
            const float ks = a.scale_log2 * exp2_int(ek0), es = (float)ev0;
            float top[T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                r[t].template hide<MASK>(sc[t], b, ks, es, add[t]);
                top[t] = r[t].template top_of<MASK>(sc[t], ks, es);
            }
            raise(r, top);
            if constexpr (T == 1) {
                kv8_f16x8 p[2];
                r[0].template weights<MASK>(sc[0], ks, es, ev0, p);
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    kv8_f16x8 y[2];
                    codes_f16x16(vc[c], y[0], y[1]);
                    vc[c] = codes_at<ONCE>(vn + v_off + c * (kBlk * 32));
                    r[0].o[c] = mfma(y[0], p[0], r[0].o[c]);
                    r[0].o[c] = mfma(y[1], p[1], r[0].o[c]);
                }
            } else {
                kv8_f16x8 y[KC][2];
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    codes_f16x16(vc[c], y[c][0], y[c][1]);
                    vc[c] = codes_at<ONCE>(vn + v_off + c * (kBlk * 32));
                }
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    kv8_f16x8 p[2];
                    r[t].template weights<MASK>(sc[t], ks, es, ev0, p);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int c = 0; c < KC; ++c) r[t].o[c] = mfma(y[c][u], p[u], r[t].o[c]);
                }
            }
        }
    }
    // the waves' results into LDS, half of the accumulators at a time, and a quarter of them out of it for each wave
    constexpr int kHalf = KC / 2, kPlace = kHalf * 4 * 64 * 4 + 64;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        r[t].l = sum_halves(r[t].l);
        int again = r0 + t * 32;
        asm volatile("" : "+s"(again));  // (the seat is looked up again: kept, it takes registers from the loop)
        seat[t] = seat_of(a, w.n, w.g, again);
        float m = kLowest, l = 0.0f, f[kWaves];
        char* row = a.out + (int64_t)seat[t].head * a.o_nb1 + (int64_t)seat[t].j * a.o_nb2 + (int64_t)w.s * a.o_nb3;
        float* part = a.part + ((int64_t)w.id * T + t) * tile_floats(D);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            __syncthreads();  // (what was there has been read)
            if (seat[t].live) {
#pragma unroll
                for (int c = 0; c < kHalf; ++c)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x16& o = r[t].o[half * kHalf + c];
                        *reinterpret_cast<kv8_f32x4*>(lds + wave * kPlace + ((c * 4 + i / 4) * 64 + lane) * 4) = kv8_f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
                    }
                if (half == 0 && h == 0) {
                    lds[wave * kPlace + kPlace - 64 + n] = r[t].m;
                    lds[wave * kPlace + kPlace - 32 + n] = r[t].l;
                }
            }
            __syncthreads();
            if (!seat[t].live) continue;
            if (half == 0) {
#pragma unroll
                for (int k = 0; k < kWaves; ++k) {
                    f[k] = lds[k * kPlace + kPlace - 64 + n];
                    m = fmaxf(m, f[k]);
                }
#pragma unroll
                for (int k = 0; k < kWaves; ++k) {
                    f[k] = __builtin_amdgcn_exp2f(f[k] - m);
                    l = fmaf(lds[k * kPlace + kPlace - 32 + n], f[k], l);
                }
            }
            const float inv = w.pieces > 1 ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
            for (int i = 0; i < kHalf; ++i) {
                const int at = wave * kHalf + i, quad = half * kHalf * 4 + at;
                kv8_f32x4 x = {};
#pragma unroll
                for (int k = 0; k < kWaves; ++k) x += *reinterpret_cast<const kv8_f32x4*>(lds + k * kPlace + (at * 64 + lane) * 4) * f[k];
                if (w.pieces > 1)
                    *reinterpret_cast<kv8_f32x4*>(part + (quad * 64 + lane) * 4) = x;
                else
                    store4(a, row, quad / 4 * 32 + quad % 4 * 8 + 4 * h, x * inv);
            }
        }
        if (seat[t].live && w.pieces > 1 && wave == 0 && h == 0) {
            part[32 * D + n] = m;
            part[32 * D + 32 + n] = l;
        }
    }
}

// N products whose left operands come from LDS: A reads first, then two more with every two products, so that a
// read has the time of A - 2 products to arrive.
template <int N, int A>
__device__ __forceinline__ void feed() {
    __builtin_amdgcn_sched_group_barrier(0x100, A, 0);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
}

// Four waves of 32 rows each over the same cells, NB blocks of 32 a step.  A wave without rows still converts
// its share of the codes: three waves of rows and one without measured faster than a work-group of three.
//
// Bound by instructions, not by memory: a wave's 32 x 32 scores and their product with V are 16 MFMAs of 32 cycles
// (128 dims) next to some 70 VALU instructions of softmax, 16 of them exponentials at a quarter of the rate, and a
// quarter of the conversions.  2048 rows behind 4096 cells, 128 dims: 178 us, 725 TFLOP/s; the matrix cores are busy
// for 28 % of the time and the VALU for 39 %, two waves of a SIMD overlap them in part, and the chunk's 384 work-groups
// leave half of the CUs with one instead of two.  96 rows of 32 streams, up to 16k cells: 99 us (2.8 TB/s).
constexpr int kStep128 = 2;  // blocks of a step
constexpr size_t kLds128 = (size_t)2 * 2 * kStep128 * (128 / 32) * 2 * 64 * 16;
template <bool MASK>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attn_rows128_kernel(Kv8AttnArgs a) {
    constexpr int D = 128, NB = kStep128, NW = kWaves;
    constexpr int KC = D / 32, ITEMS = NB * KC, MINE = ITEMS / NW;
    constexpr int kAhead = 6;  // LDS reads ahead of their products
    static_assert(ITEMS % NW == 0, "every wave converts the same share");
    extern __shared__ __align__(16) float lds[];
    // [buffer][K, V][block, piece][first, second eight][lane] 8 f16
    typedef kv8_f16x8 Tile[2][ITEMS][2][64];
    Tile* tile = reinterpret_cast<Tile*>(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!work_of(a, w)) return;
    const int r0 = w.tile * (32 * NW);
    int mine = r0 + wave * 32;
    Seat seat = seat_of(a, w.n, w.g, mine);
    Rows<D> one[1], &r = one[0];
    r.begin(a, w.n, mine, seat);
    kv8_f16x8 q[KC][2];
#pragma unroll
    for (int c = 0; c < KC; ++c) Rows<D>::queries(a, w.s, seat, c, q[c]);
    const char* mask = MASK ? a.mask + (int64_t)seat.j * a.m_nb1 + (int64_t)w.s * a.m_nb3 : nullptr;
    int last = w.last;  // blocks that any row of the work-group sees
    if (a.mode == SIXI_MASK_BLOCK_CAUSAL)
        last = min(last, (w.n.cached + (min(r0 + 32 * NW, w.n.rows * a.G) - 1) / a.G + kBlk) / kBlk);
    if (w.first < last) {
        kv8_u32x4 codes[2][MINE];  // the wave's share of the next step's, on their way
        int ek[NB], ev[NB];
        BlockWalk walk;
        // the walk's step; a second block that is none is the first once more (its cells are hidden).  The
        // compiler is not to know that: it would wait for the first one's exponents to copy them.
        auto load = [&](int which) {
            const bool both = walk.b + 1 < last;
            int step = both ? (which ? walk.v_nb : walk.k_nb) : 0;
            asm("" : "+s"(step));
            const char* p = which ? walk.v : walk.k;
            const int n = lane & 31, h = lane >> 5;
            const uint32_t off = which ? n * kBlk + h * 16 : h * (kBlk * 16) + (16 * (n / 4 % 2) + 4 * (n / 8) + n % 4) * 16;
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const int it = wave + i * NW;
                codes[which][i] = *reinterpret_cast<const kv8_u32x4*>(p + ((it >= KC ? step : 0) + it % KC * (kBlk * 32)) + off);
            }
        };
        auto load_exps = [&]() {
            const bool both = walk.b + 1 < last;
            int ke_step = both ? walk.ke_nb : 0, ve_step = both ? walk.ve_nb : 0;
            asm("" : "+s"(ke_step), "+s"(ve_step));
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                ek[i] = walk.ke[i * ke_step];
                ev[i] = walk.ve[i * ve_step];
            }
        };
        float ks[NB], es[NB];
        int e0[NB];
        // codes as f16 into a buffer
        auto convert = [&](int buf, int which) {
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                kv8_f16x8 x, y;
                codes_f16x16(codes[which][i], x, y);
                tile[buf][which][wave + i * NW][0][lane] = x;
                tile[buf][which][wave + i * NW][1][lane] = y;
            }
        };
        auto scales = [&]() {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                ks[i] = a.scale_log2 * exp2_int(clamp_exp(ek[i]));
                e0[i] = clamp_exp(ev[i]);
                es[i] = (float)e0[i];
            }
        };
        // One step.  The products run at a raised priority, so that the matrix cores serve one wave of a SIMD
        // while the other is at its softmax.
        auto step = [&](int b, auto BUF) {
            constexpr int buf = decltype(BUF)::value;
            const bool any = b * kBlk < r.reach;
            f32x16 sc[NB] = {};
            // (behind the last step: its blocks once more, and not used)
            load(0);
            load(1);
            load_exps();
            walk.go(a.pages, a.k, a.v, w.s, w.g, NB);
            f16x8u add[NB][2];
            if (any) {
                if (MASK)
#pragma unroll
                    for (int i = 0; i < NB; ++i) Rows<D>::mask_of(mask, min(b + i, last - 1), add[i]);
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < NB; ++i) sc[i] = mfma(tile[buf][0][i * KC + c][u][lane], q[c][u], sc[i]);
                feed<2 * NB * KC, kAhead>();
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (any) {
                kv8_f16x8 p[NB][2];
                float top[1] = {kLowest};
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    r.template hide<MASK>(sc[i], b + i, ks[i], es[i], add[i]);
                    top[0] = __builtin_elementwise_maximum(top[0], r.template top_of<MASK>(sc[i], ks[i], es[i]));
                }
                raise(one, top);
#pragma unroll
                for (int i = 0; i < NB; ++i) r.template weights<MASK>(sc[i], ks[i], es[i], e0[i], p[i]);
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int c = 0; c < KC; ++c) r.o[c] = mfma(tile[buf][1][i * KC + c][u][lane], p[i][u], r.o[c]);
                feed<2 * NB * KC, kAhead>();
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            }
            convert(buf ^ 1, 0);
            convert(buf ^ 1, 1);
            scales();
            __syncthreads();
        };
        walk.begin(a.pages, a.k, a.v, w.s, w.g, w.first, last);
        load(0);
        load_exps();
        convert(0, 0);
        load(1);
        convert(0, 1);
        scales();
        walk.go(a.pages, a.k, a.v, w.s, w.g, NB);
        __syncthreads();
        // steps in pairs, one for each buffer.  (A loop of its own for the steps whose cells every row sees took
        // 50 more registers, and with them the reads ahead: 203 against 182 us for the prompt chunk.)
        using std::integral_constant;
#pragma unroll 1
        for (int b = w.first; b < last; b += 2 * NB) {
            step(b, integral_constant<int, 0>{});
            if (b + NB < last) step(b + NB, integral_constant<int, 1>{});
        }
    }
    r.l = sum_halves(r.l);
    asm volatile("" : "+s"(mine));  // (the seat is looked up again: kept, it takes registers from the loop)
    seat = seat_of(a, w.n, w.g, mine);
    if (w.pieces == 1)
        r.finish(a, w.s, seat);
    else
        r.leave(a.part + ((int64_t)w.id * NW + wave) * tile_floats(D), seat);
}

// The same at 256 dims, where accumulators and queries leave few registers: most of the queries in LDS, K and V one
// buffer each, a block a step with two barriers: V becomes f16 beside the scores' products and the next K beside the
// output's, so that both have their codes on the way for a whole step and nothing is left in scratch memory.
//
// Bound as at 128 dims, with a barrier for every 16 MFMAs.  Trees of 12 tokens, 8 streams of 2k to 9k cells: 50 us, and
// 55 with the queries in registers, two buffers and one tensor's codes on their way (2 streams up to 50k cells 69 and
// 79); 16 tokens of 16 streams up to 16k cells 99 and 102; 1024 rows behind 2048 cells 119 and 115; 173 rows
// behind 11400 cells 79 to 80 us, 610 TFLOP/s, and 79.  Where rows are cut their f32 partial results cost as much again as
// the codes: the merge is 13 us of the last.
constexpr int kKept256 = 2;  // pieces of the queries in registers
struct Lds256 {
    kv8_f16x8 k[8][2][64], v[8][2][64];   // [piece][first, second eight][lane]
    kv8_f16x8 q[kWaves][8 - kKept256][2][64];   // what a wave's registers do not keep of its queries
};

template <bool MASK>
__global__ __launch_bounds__(kWaves * 64, 2) void kv8_attn_rows256_kernel(Kv8AttnArgs a) {
    constexpr int D = 256, KC = D / 32, MINE = KC / kWaves, kKept = kKept256;
    extern __shared__ __align__(16) float lds[];
    Lds256& x = *reinterpret_cast<Lds256*>(lds);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Work w;
    if (!work_of(a, w)) return;
    const int r0 = w.tile * (32 * kWaves);
    int mine = r0 + wave * 32;
    Seat seat = seat_of(a, w.n, w.g, mine);
    Rows<D> one[1], &r = one[0];
    r.begin(a, w.n, mine, seat);
    kv8_f16x8 q[kKept][2];
#pragma unroll
    for (int c = 0; c < kKept; ++c) Rows<D>::queries(a, w.s, seat, c, q[c]);
#pragma unroll
    for (int c = kKept; c < KC; ++c) {
        kv8_f16x8 y[2];
        Rows<D>::queries(a, w.s, seat, c, y);
        x.q[wave][c - kKept][0][lane] = y[0];
        x.q[wave][c - kKept][1][lane] = y[1];
    }
    const char* masks = MASK ? a.mask + (int64_t)w.s * a.m_nb3 : nullptr;
    const int j = seat.j;
    int last = w.last;  // blocks that any row of the work-group sees
    if (a.mode == SIXI_MASK_BLOCK_CAUSAL)
        last = min(last, (w.n.cached + (min(r0 + 32 * kWaves, w.n.rows * a.G) - 1) / a.G + kBlk) / kBlk);
    if (w.first < last) {
        kv8_u32x4 kc[MINE], vc[MINE];
        int ek, ev, e0;
        float ks, es;
        BlockWalk walk;
        // (offsets are formed again at each use: kept, they take registers)
        auto load_k = [&]() {
            int at = lane;
            asm volatile("" : "+v"(at));
            const int n = at & 31, h = at >> 5;
            const uint32_t off = h * (kBlk * 16) + (16 * (n / 4 % 2) + 4 * (n / 8) + n % 4) * 16;
#pragma unroll
            for (int i = 0; i < MINE; ++i) kc[i] = *reinterpret_cast<const kv8_u32x4*>(walk.k + (wave + i * kWaves) * (kBlk * 32) + off);
            ek = *walk.ke;
            ev = *walk.ve;
        };
        auto load_v = [&]() {
            int at = lane;
            asm volatile("" : "+v"(at));
            const uint32_t off = (at & 31) * kBlk + (at >> 5) * 16;
#pragma unroll
            for (int i = 0; i < MINE; ++i) vc[i] = *reinterpret_cast<const kv8_u32x4*>(walk.v + (wave + i * kWaves) * (kBlk * 32) + off);
        };
        auto convert = [&](const kv8_u32x4 (&codes)[MINE], kv8_f16x8 (&to)[8][2][64]) {
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                kv8_f16x8 lo, hi;
                codes_f16x16(codes[i], lo, hi);
                to[wave + i * kWaves][0][lane] = lo;
                to[wave + i * kWaves][1][lane] = hi;
            }
        };
        auto scales = [&]() {
            ks = a.scale_log2 * exp2_int(clamp_exp(ek));
            e0 = clamp_exp(ev);
            es = (float)e0;
        };
        // (a scalar, so that branches on it are: waits for loads would count those of a path that no wave takes)
        const int reach = __builtin_amdgcn_readfirstlane(r.reach);
        walk.begin(a.pages, a.k, a.v, w.s, w.g, w.first, last);
        load_k();
        load_v();
        convert(kc, x.k);
        scales();
        walk.go(a.pages, a.k, a.v, w.s, w.g, 1);
        load_k();
        __syncthreads();
#pragma unroll 1
        for (int b = w.first; b < last; ++b) {
            const bool any = b * kBlk < reach;
            f16x8u add[2];
            kv8_f16x8 p[2];
            f32x16 sc[1] = {};
            if (any) {
                if (MASK) {
                    int row = j;
                    asm volatile("" : "+v"(row));
                    Rows<D>::mask_of(masks + (int64_t)row * a.m_nb1, b, add);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        sc[0] = mfma(x.k[c][u][lane], c < kKept ? q[c < kKept ? c : 0][u] : x.q[wave][c < kKept ? 0 : c - kKept][u][lane], sc[0]);
                convert(vc, x.v);
                __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
                for (int i = 0; i < 2 * kKept - 3; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
                }
#pragma unroll
                for (int i = 2 * kKept - 3; i < 2 * KC; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                convert(vc, x.v);
            }
            load_v();  // (in one place: where two paths load, the registers are copied, which waits for them)
            if (any) {
                r.template hide<MASK>(sc[0], b, ks, es, add);
                const float top[1] = {r.template top_of<MASK>(sc[0], ks, es)};
                raise(one, top);
                r.template weights<MASK>(sc[0], ks, es, e0, p);
            }
            scales();
            walk.go(a.pages, a.k, a.v, w.s, w.g, 1);
            __syncthreads();
            if (any) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int c = 0; c < KC; ++c) r.o[c] = mfma(x.v[c][u][lane], p[u], r.o[c]);
                convert(kc, x.k);
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                for (int i = 0; i < 2 * KC; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
            } else {
                convert(kc, x.k);
            }
            load_k();
            __syncthreads();
        }
    }
    r.l = sum_halves(r.l);
    asm volatile("" : "+s"(mine));  // (the seat is looked up again: kept, it takes registers from the loop)
    seat = seat_of(a, w.n, w.g, mine);
    if (w.pieces == 1)
        r.finish(a, w.s, seat);
    else
        r.leave(a.part + ((int64_t)w.id * kWaves + wave) * tile_floats(D), seat);
}

// Joins the pieces of 32 rows: D/32 work-groups of four waves, each with 4 of the accumulators' D/8 quads.  What a
// call's pieces left was written on other XCDs and comes from memory, so everything a wave needs is asked for at
// once: up to 8 pieces by a wave for each quad, more by all four waves for all four quads, joined in LDS.
template <int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8AttnArgs a) {
    __shared__ __align__(16) kv8_f32x4 sums[kWaves][4][64];
    __shared__ float tops[kWaves][32], totals[kWaves][32];
    const int s = blockIdx.z, g = blockIdx.y, quads = blockIdx.x % (D / 32), t32 = blockIdx.x / (D / 32);
    const Place p = a.places[s];  // (asked for with the lengths: a stream without rows has left none, and reads none)
    const Lens len = lens_of(a, s);
    const int M = len.rows * a.G;
    if (t32 * 32 >= M || p.pieces == 1) return;
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quad = quads * 4 + wave, rr = t32 * 32 + n;
    const bool live = rr < M;
    const int64_t step = (int64_t)a.Hkv * a.waves * tile_floats(D);  // from piece to piece
    const float* at = a.part + (((int64_t)p.at + (int64_t)(p.tiles - 1 - t32 / a.waves) * p.pieces * a.Hkv + g) * a.waves + t32 % a.waves) * tile_floats(D);
    float m = kLowest, l = 0.0f;
    kv8_f32x4 o = {};
    if (p.pieces <= 8) {
        float ms[8], ls[8];
        kv8_f32x4 os[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool on = live && i < p.pieces;
            ms[i] = on ? at[i * step + 32 * D + n] : kLowest;
            ls[i] = on ? at[i * step + 32 * D + 32 + n] : 0.0f;
            os[i] = on ? *reinterpret_cast<const kv8_f32x4*>(at + i * step + (quad * 64 + lane) * 4) : kv8_f32x4{};
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, ms[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = __builtin_amdgcn_exp2f(ms[i] - m);
            l = fmaf(ls[i], f, l);
            o += os[i] * f;
        }
    } else {
        kv8_f32x4 x[4] = {};
        for (int i0 = wave; i0 < p.pieces; i0 += 4 * kWaves) {
            float ms[4], ls[4];
            kv8_f32x4 os[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * kWaves;
                const bool on = live && i < p.pieces;
                ms[k] = on ? at[i * step + 32 * D + n] : kLowest;
                ls[k] = on ? at[i * step + 32 * D + 32 + n] : 0.0f;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    os[k][q] = on ? *reinterpret_cast<const kv8_f32x4*>(at + i * step + ((quads * 4 + q) * 64 + lane) * 4) : kv8_f32x4{};
            }
            const float up = fmaxf(fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3])), m), f0 = __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= f0;
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] *= f0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = __builtin_amdgcn_exp2f(ms[k] - m);
                l = fmaf(ls[k], f, l);
#pragma unroll
                for (int q = 0; q < 4; ++q) x[q] += os[k][q] * f;
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[wave][q][lane] = x[q];
        if (h == 0) {
            tops[wave][n] = m;
            totals[wave][n] = l;
        }
        __syncthreads();
        m = kLowest;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) m = fmaxf(m, tops[k][n]);
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            const float f = __builtin_amdgcn_exp2f(tops[k][n] - m);
            l = fmaf(totals[k][n], f, l);
            o += sums[k][wave][lane] * f;
        }
    }
    if (!live) return;
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    const int j = rr / a.G, head = g * a.G + rr % a.G;
    store4(a, a.out + (int64_t)head * a.o_nb1 + (int64_t)j * a.o_nb2 + (int64_t)s * a.o_nb3, quad / 4 * 32 + quad % 4 * 8 + 4 * h, o * inv);
}

template <int D, int T, bool MASK>
void launch_few(const Kv8AttnArgs& a, hipStream_t stream) {
    constexpr size_t lds = (size_t)kWaves * (16 * D + 64) * sizeof(float);
    static_assert(lds >= (size_t)T * (D / 32) * 2 * 64 * 16, "the queries lie where the results are joined");
    if (a.once)
        hipLaunchKernelGGL((kv8_attn_few_kernel<D, T, MASK, true>), dim3((unsigned)a.grid), dim3(kWaves * 64), lds, stream, a);
    else
        hipLaunchKernelGGL((kv8_attn_few_kernel<D, T, MASK, false>), dim3((unsigned)a.grid), dim3(kWaves * 64), lds, stream, a);
}
template <int D, bool MASK>
void launch_pieces(const Kv8AttnArgs& a, hipStream_t stream) {
    if (a.waves == 1) return launch_few<D, 1, MASK>(a, stream);
    if constexpr (D == 128 && !MASK)
        if (a.waves == 2) return launch_few<D, 2, MASK>(a, stream);
    if constexpr (D == 128)
        hipLaunchKernelGGL(kv8_attn_rows128_kernel<MASK>, dim3((unsigned)a.grid), dim3(kWaves * 64), kLds128, stream, a);
    else
        hipLaunchKernelGGL(kv8_attn_rows256_kernel<MASK>, dim3((unsigned)a.grid), dim3(kWaves * 64), sizeof(Lds256), stream, a);
}

template <int D>
hipError_t launch(const Kv8AttnArgs& a, hipStream_t stream) {
    if (a.mode == SIXI_MASK_EXPLICIT)
        launch_pieces<D, true>(a, stream);
    else
        launch_pieces<D, false>(a, stream);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.cut) return e;
    // (a cut stream has fewer tiles than make 3/4 of the target over the heads)
    const int64_t t32 = std::min(((int64_t)a.n_q * a.G + 31) / 32, (3 * (int64_t)a.target / (4 * a.Hkv) + 1) * a.waves);
    hipLaunchKernelGGL(kv8_merge_kernel<D>, dim3((unsigned)(t32 * (D / 32)), (unsigned)a.Hkv, (unsigned)a.S), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace

size_t kv8_attn_plan(Kv8AttnArgs& a) {
    const int64_t t32 = ((int64_t)a.n_q * a.G + 31) / 32;
    // 33 to 64 rows of 128 dims: both tiles in every wave's registers, where two of the rows kernel's four waves
    // would only convert (32 streams of 48 rows, up to 16k cells: 70 against 95 us).  Not with a mask: its values
    // do not fit beside them (32 streams of 60 rows: 175 against 118 us).
    const bool two = t32 == 2 && a.D == 128 && a.mode != SIXI_MASK_EXPLICIT;
    a.waves = t32 == 1 ? 1 : two ? 2 : kWaves;
    a.target = 2 * device_cu_count();  // (two work-groups on a CU)
    // Codes that the 256 MB behind the L2 cannot hold until the next call go past it, where one work-group reads each
    // (a token of 32 streams, 269 MB: 53 against 61 us; 8 streams of 256 dims, 320 MB: 66 against 73).  Fewer may
    // still be there (one stream of 50k cells, 102 MB, called in turn with another: 38 against 35 the other way), and
    // where several tiles read them, or the rows kernels, they are better kept (96 rows: 104 against 99).
    a.once = a.code_bytes >= (int64_t)256 << 20;
    a.least = 4;
    const int64_t tiles = (t32 + a.waves - 1) / a.waves * a.Hkv * a.S;
    const int64_t blocks = (a.n_kv + kBlk - 1) / kBlk;
    // pieces at most: one for each tile, and those that a cut makes (the last few: the round-robin over 8
    // XCDs, and f32 sums of large numbers); a cut is made only over fewer tiles than 3/4 of the target
    // (none where the host can tell that the tiles are enough: then there is nothing to join)
    a.cut = blocks > a.least && (a.q_len || !enough(tiles / a.Hkv, a));
    a.grid = (int32_t)(tiles + (a.cut ? a.target : 0) + 16);
    if (!a.cut) return 256;
    const int64_t slots = (tiles < a.target ? tiles : a.target) + a.target + 16;
    if (a.part) a.places = reinterpret_cast<Kv8Place*>(a.part + slots * a.waves * tile_floats(a.D));
    return ((size_t)slots * a.waves * tile_floats(a.D) * sizeof(float) + (size_t)a.S * sizeof(Kv8Place) + 255) / 256 * 256;
}

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t stream) {
    return a.D == 128 ? launch<128>(a, stream) : launch<256>(a, stream);
}

}  // namespace sixi
