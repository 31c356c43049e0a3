// sixi_kv8_abi.cpp -- the C ABI of include/sixi_kv8.h: validation on the host, the kernels in
// kv8_store.hip and kv8_attn.hip.
//
// As in sixi_attn_abi.cpp every error is a status (the reference's ErrorCode values of
// include/sixi_asi/common.hpp:40-67, negated).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "abi_util.hpp"
#include "kv8_internal.hpp"
#include "sixi_kv8.h"

namespace {

using namespace sixi_abi;

constexpr int64_t kPageRow = (int64_t)1 << 26;  // cells of a stream

// A tensor of blocks as a view: [bytes of a block, blocks, heads, streams or pages].
sixi_view block_view(const void* data, const int64_t (&nb)[3], int64_t block_bytes, const sixi_kv8_cache& c) {
    sixi_view v{};
    v.data = data;
    v.ne[0] = block_bytes;
    v.ne[1] = c.n_blocks;
    v.ne[2] = c.n_heads;
    v.ne[3] = c.n;
    v.nb[0] = 1;
    for (int i = 0; i < 3; ++i) v.nb[1 + i] = nb[i];
    return v;
}

struct CacheViews {
    sixi_view k, v, ke, ve;
};

int check_cache(const sixi_kv8_cache& c, bool paged, CacheViews* out) {
    if (!c.k || !c.v || !c.k_exp || !c.v_exp) return SIXI_E_INVALID_ARGUMENT;
    if (c.n_heads <= 0 || c.n_blocks <= 0 || c.n <= 0) return SIXI_E_INVALID_ARGUMENT;
    if (c.head_dim != 128 && c.head_dim != 256) return SIXI_E_UNSUPPORTED;
    if (paged && c.n_blocks != sixi::kPageBlocks) return SIXI_E_INVALID_ARGUMENT;
    if (c.n > INT32_MAX || c.n_heads > 4096 || c.n_blocks > kPageRow / sixi::kBlk) return SIXI_E_UNSUPPORTED;
    for (int i = 0; i < 3; ++i) {
        if (c.k_nb[i] < 0 || c.v_nb[i] < 0 || c.k_exp_nb[i] < 0 || c.v_exp_nb[i] < 0) return SIXI_E_INVALID_ARGUMENT;
        if (c.k_nb[i] % 16 || c.v_nb[i] % 16) return SIXI_E_ALIGNMENT;
        const int64_t most = INT32_MAX / 2;  // (steps from block to block are 32-bit)
        if (i == 0 && (c.k_nb[0] > most || c.v_nb[0] > most || c.k_exp_nb[0] > most || c.v_exp_nb[0] > most)) return SIXI_E_UNSUPPORTED;
    }
    if (!aligned(c.k, 16) || !aligned(c.v, 16)) return SIXI_E_ALIGNMENT;
    const int64_t bytes = (int64_t)sixi::kBlk * c.head_dim;
    out->k = block_view(c.k, c.k_nb, bytes, c);
    out->v = block_view(c.v, c.v_nb, bytes, c);
    out->ke = block_view(c.k_exp, c.k_exp_nb, 1, c);
    out->ve = block_view(c.v_exp, c.v_exp_nb, 1, c);
    for (const sixi_view* v : {&out->k, &out->v, &out->ke, &out->ve}) {
        if (view_span(*v, v->ne[0]) < 0) return SIXI_E_INTEGER_OVERFLOW;
        if (!rows_disjoint(*v, v->ne[0])) return SIXI_E_INVALID_ARGUMENT;
    }
    return SIXI_OK;
}

int check_pages(const int32_t* pt, int64_t stride, int64_t* blocks) {
    if (!pt) return SIXI_OK;
    if (stride <= 0 || stride > kPageRow / SIXI_KV_PAGE_CELLS) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(pt, 4)) return SIXI_E_ALIGNMENT;
    *blocks = stride * sixi::kPageBlocks;
    return SIXI_OK;
}

sixi::Kv8Tensor tensor_of(void* codes, int8_t* exps, const int64_t (&nb)[3], const int64_t (&e_nb)[3]) {
    sixi::Kv8Tensor t{};
    t.codes = static_cast<char*>(codes);
    t.exps = exps;
    for (int i = 0; i < 3; ++i) {
        t.nb[i] = nb[i];
        t.e_nb[i] = e_nb[i];
    }
    return t;
}

// Whether a written range meets the lengths or the page table.
template <typename P>
bool meets_arrays(const void* w, int64_t bytes, const P& p, int64_t S) {
    return (p.kv_len && ranges_overlap(w, bytes, p.kv_len, S * 4)) || (p.q_len && ranges_overlap(w, bytes, p.q_len, S * 4)) ||
           (p.page_table && ranges_overlap(w, bytes, p.page_table, S * p.page_table_stride * 4));
}

int resolve_rows(const sixi_kv8_rows_params* p, bool read, sixi::Kv8RowsArgs* out) {
    if (!p || p->flags != 0) return SIXI_E_INVALID_ARGUMENT;
    const sixi_kv8_cache& c = p->cache;
    const bool paged = p->page_table != nullptr;
    CacheViews cv{};
    int rc = check_cache(c, paged, &cv);
    if (rc != SIXI_OK) return rc;
    int64_t blocks = c.n_blocks;
    rc = check_pages(p->page_table, p->page_table_stride, &blocks);
    if (rc != SIXI_OK) return rc;
    const int64_t D = c.head_dim, n_rows = p->k.ne[1], S = p->k.ne[3];
    sixi::Kv8RowsArgs a{};
    const sixi_view* rows[2] = {&p->k, &p->v};
    for (int i = 0; i < 2; ++i) {
        const sixi_view& r = *rows[i];
        const int es = elem_bytes(r.type);
        if (es == 0 || r.nb[0] != es) return SIXI_E_INVALID_ARGUMENT;
        if (r.ne[0] != D || r.ne[1] != n_rows || r.ne[2] != c.n_heads || r.ne[3] != S) return SIXI_E_INVALID_ARGUMENT;
        if (n_rows < 0 || S < 0 || (!r.data && n_rows > 0 && S > 0)) return SIXI_E_INVALID_ARGUMENT;
        if (n_rows > kPageRow) return SIXI_E_INTEGER_OVERFLOW;
        for (int d = 1; d < 4; ++d) {
            if (r.nb[d] < 0) return SIXI_E_INVALID_ARGUMENT;
            if (r.nb[d] % 16) return SIXI_E_ALIGNMENT;
        }
        if (!aligned(r.data, 16)) return SIXI_E_ALIGNMENT;
        const int64_t rb = D * es;
        if (view_span(r, rb) < 0) return SIXI_E_INTEGER_OVERFLOW;
        if (read && view_span(r, rb) > 0 && (!rows_disjoint(r, rb) || meets_arrays(r.data, view_span(r, rb), *p, S))) return SIXI_E_INVALID_ARGUMENT;
        for (const sixi_view* v : {&cv.k, &cv.v, &cv.ke, &cv.ve})
            if (views_overlap(r, rb, *v, v->ne[0])) return SIXI_E_INVALID_ARGUMENT;
        a.rows[i] = static_cast<char*>(const_cast<void*>(r.data));
        a.r_nb1[i] = r.nb[1];
        a.r_nb2[i] = r.nb[2];
        a.r_nb3[i] = r.nb[3];
        a.f16[i] = r.type == SIXI_TYPE_F16;
    }
    if (S > 65535) return SIXI_E_UNSUPPORTED;
    if (!paged && c.n != S) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(p->kv_len, 4) || !aligned(p->q_len, 4)) return SIXI_E_ALIGNMENT;
    if (read) {
        if (views_overlap(p->k, D * elem_bytes(p->k.type), p->v, D * elem_bytes(p->v.type))) return SIXI_E_INVALID_ARGUMENT;
    } else {
        // four tensors written by different work-groups
        const sixi_view* w[4] = {&cv.k, &cv.v, &cv.ke, &cv.ve};
        for (int i = 0; i < 4; ++i) {
            for (int j = i + 1; j < 4; ++j)
                if (views_overlap(*w[i], w[i]->ne[0], *w[j], w[j]->ne[0])) return SIXI_E_INVALID_ARGUMENT;
            if (meets_arrays(w[i]->data, view_span(*w[i], w[i]->ne[0]), *p, S)) return SIXI_E_INVALID_ARGUMENT;
        }
    }
    a.t[0] = tensor_of(c.k, c.k_exp, c.k_nb, c.k_exp_nb);
    a.t[1] = tensor_of(c.v, c.v_exp, c.v_nb, c.v_exp_nb);
    a.pages = {p->page_table, p->page_table_stride, (int32_t)c.n, (int32_t)blocks};
    a.kv_len = p->kv_len;
    a.q_len = p->q_len;
    a.D = (int32_t)D;
    a.n_rows = (int32_t)n_rows;
    a.Hkv = c.n_heads;
    a.S = (int32_t)S;
    *out = a;
    return SIXI_OK;
}

int resolve_attn(const sixi_kv8_attn_params* p, sixi::Kv8AttnArgs* out, size_t* ws) {
    if (!p || p->flags != 0) return SIXI_E_INVALID_ARGUMENT;
    const sixi_kv8_cache& c = p->cache;
    const bool paged = p->page_table != nullptr;
    const sixi_view &q = p->q, &o = p->out;
    if (!q.data || !o.data) return SIXI_E_INVALID_ARGUMENT;
    CacheViews cv{};
    int rc = check_cache(c, paged, &cv);
    if (rc != SIXI_OK) return rc;
    int64_t blocks = c.n_blocks;
    rc = check_pages(p->page_table, p->page_table_stride, &blocks);
    if (rc != SIXI_OK) return rc;
    const int qes = elem_bytes(q.type), oes = elem_bytes(o.type);
    if (qes == 0 || oes == 0) return SIXI_E_UNSUPPORTED;
    for (int d = 0; d < 4; ++d)
        if (q.ne[d] <= 0 || o.ne[d] <= 0 || q.nb[d] < 0 || o.nb[d] < 0) return SIXI_E_INVALID_ARGUMENT;
    const int64_t D = c.head_dim, n_q = q.ne[1], H = q.ne[2], S = q.ne[3], n_kv = blocks * sixi::kBlk;
    if (q.ne[0] != D || H % c.n_heads != 0) return SIXI_E_INVALID_ARGUMENT;
    if (o.ne[0] != D || o.ne[1] != H || o.ne[2] != n_q || o.ne[3] != S) return SIXI_E_INVALID_ARGUMENT;
    if (!paged && c.n != S) return SIXI_E_INVALID_ARGUMENT;
    if (S > 512 || H > 4096 || n_q > (1 << 20)) return SIXI_E_UNSUPPORTED;
    if (q.nb[0] != qes || o.nb[0] != oes) return SIXI_E_INVALID_ARGUMENT;
    for (int d = 1; d < 4; ++d)
        if (q.nb[d] % 16 || o.nb[d] % 16) return SIXI_E_ALIGNMENT;
    if (!aligned(q.data, 16) || !aligned(o.data, 16) || !aligned(p->kv_len, 4) || !aligned(p->q_len, 4)) return SIXI_E_ALIGNMENT;
    const int64_t qb = D * qes, ob = D * oes;
    if (view_span(q, qb) < 0 || view_span(o, ob) < 0) return SIXI_E_INTEGER_OVERFLOW;
    // work-groups write output rows in no fixed order, while others read
    if (!rows_disjoint(o, ob) || views_overlap(o, ob, q, qb)) return SIXI_E_INVALID_ARGUMENT;
    for (const sixi_view* v : {&cv.k, &cv.v, &cv.ke, &cv.ve})
        if (views_overlap(o, ob, *v, v->ne[0])) return SIXI_E_INVALID_ARGUMENT;
    if (meets_arrays(o.data, view_span(o, ob), *p, S)) return SIXI_E_INVALID_ARGUMENT;

    const int mode = p->mask_mode;
    if (mode < SIXI_MASK_NONE || mode > SIXI_MASK_EXPLICIT) return SIXI_E_INVALID_ARGUMENT;
    if (mode == SIXI_MASK_BLOCK_CAUSAL && !p->kv_len) return SIXI_E_INVALID_ARGUMENT;
    if (p->kv_len && n_q > n_kv) return SIXI_E_INVALID_ARGUMENT;
    const sixi_view& m = p->mask;
    if (mode == SIXI_MASK_EXPLICIT) {
        if (!m.data || m.type != SIXI_TYPE_F16 || m.nb[0] != 2) return SIXI_E_INVALID_ARGUMENT;
        if (m.ne[0] < n_kv || m.ne[1] < n_q || m.ne[2] != 1 || (m.ne[3] != 1 && m.ne[3] != S)) return SIXI_E_INVALID_ARGUMENT;
        if (m.nb[1] < 0 || m.nb[3] < 0) return SIXI_E_INVALID_ARGUMENT;
        if (m.nb[1] % 2 || m.nb[3] % 2 || !aligned(m.data, 2)) return SIXI_E_ALIGNMENT;
        if (view_span(m, m.ne[0] * 2) < 0) return SIXI_E_INTEGER_OVERFLOW;
        if (views_overlap(o, ob, m, m.ne[0] * 2)) return SIXI_E_INVALID_ARGUMENT;
    }
    // (2^40 over every scale in range stays within f32)
    if (!(std::fabs(p->scale) <= 0x1p40f)) return SIXI_E_INVALID_ARGUMENT;

    sixi::Kv8AttnArgs a{};
    a.q = static_cast<const char*>(q.data);
    a.q_nb1 = q.nb[1];
    a.q_nb2 = q.nb[2];
    a.q_nb3 = q.nb[3];
    a.q_f16 = q.type == SIXI_TYPE_F16;
    a.out = static_cast<char*>(const_cast<void*>(o.data));
    a.o_nb1 = o.nb[1];
    a.o_nb2 = o.nb[2];
    a.o_nb3 = o.nb[3];
    a.o_f16 = o.type == SIXI_TYPE_F16;
    a.k = tensor_of(c.k, c.k_exp, c.k_nb, c.k_exp_nb);
    a.v = tensor_of(c.v, c.v_exp, c.v_nb, c.v_exp_nb);
    a.pages = {p->page_table, p->page_table_stride, (int32_t)c.n, (int32_t)blocks};
    a.kv_len = p->kv_len;
    a.q_len = p->q_len;
    if (mode == SIXI_MASK_EXPLICIT) {
        a.mask = static_cast<const char*>(m.data);
        a.m_nb1 = m.nb[1];
        a.m_nb3 = m.ne[3] == 1 ? 0 : m.nb[3];
    }
    a.mode = mode;
    a.S = (int32_t)S;
    a.H = (int32_t)H;
    a.Hkv = c.n_heads;
    a.G = (int32_t)(H / c.n_heads);
    a.n_q = (int32_t)n_q;
    a.n_kv = (int32_t)n_kv;
    a.D = (int32_t)D;
    // a scale of 0 becomes one that no score can notice: hidden cells are -inf times it
    a.scale_log2 = std::fmax(std::fabs(p->scale) * 1.4426950408889634f, 0x1p-85f);
    a.q_sign = std::signbit(p->scale) ? -1.0f : 1.0f;
    if ((a.n_q * (int64_t)a.G + 31) / 32 * a.Hkv * S > ((int64_t)1 << 23)) return SIXI_E_UNSUPPORTED;  // work-groups
    // (pages that streams share are there once)
    a.code_bytes = (paged ? std::min(S * blocks, c.n * sixi::kPageBlocks) : S * blocks) * sixi::kBlk * D * 2 * c.n_heads;
    a.part = static_cast<float*>(p->workspace);
    *ws = sixi::kv8_attn_plan(a);
    *out = a;
    return SIXI_OK;
}

}  // namespace

extern "C" {

int sixi_kv8_rows_validate(const sixi_kv8_rows_params* p, int read) {
    sixi::Kv8RowsArgs a;
    return resolve_rows(p, read != 0, &a);
}

int sixi_kv8_write(const sixi_kv8_rows_params* p) {
    sixi::Kv8RowsArgs a;
    const int rc = resolve_rows(p, false, &a);
    if (rc != SIXI_OK) return rc;
    return sixi::launch_kv8_write(a, static_cast<hipStream_t>(p->stream)) == hipSuccess ? SIXI_OK : SIXI_E_BACKEND;
}

int sixi_kv8_read(const sixi_kv8_rows_params* p) {
    sixi::Kv8RowsArgs a;
    const int rc = resolve_rows(p, true, &a);
    if (rc != SIXI_OK) return rc;
    return sixi::launch_kv8_read(a, static_cast<hipStream_t>(p->stream)) == hipSuccess ? SIXI_OK : SIXI_E_BACKEND;
}

int sixi_kv8_pool_attach(sixi_kv_pool* pool, const sixi_kv8_cache* c) {
    if (!pool || !c) return SIXI_E_INVALID_ARGUMENT;
    CacheViews cv{};
    int rc = check_cache(*c, true, &cv);
    if (rc != SIXI_OK) return rc;
    // a head's 8 blocks as 256 rows of D bytes, its 8 exponents as one row of 8
    const int64_t block = (int64_t)sixi::kBlk * c->head_dim;
    if (c->k_nb[0] != block || c->v_nb[0] != block || c->k_exp_nb[0] != 1 || c->v_exp_nb[0] != 1) return SIXI_E_INVALID_ARGUMENT;
    sixi_view views[4];
    const sixi_view* from[4] = {&cv.k, &cv.v, &cv.ke, &cv.ve};
    for (int i = 0; i < 4; ++i) {
        views[i] = *from[i];
        views[i].type = sixi_abi::kRawBytes;
        views[i].ne[0] = i < 2 ? block * sixi::kPageBlocks : sixi::kPageBlocks;
        views[i].ne[1] = 1;
        views[i].nb[1] = views[i].ne[0];
        if (views[i].nb[2] % 2 || views[i].nb[3] % 2 || !aligned(views[i].data, 2)) return SIXI_E_ALIGNMENT;
    }
    return sixi_abi::pool_attach_raw(pool, views, 4);
}

int sixi_kv8_attn_validate(const sixi_kv8_attn_params* p) {
    sixi::Kv8AttnArgs a;
    size_t ws;
    return resolve_attn(p, &a, &ws);
}

int sixi_kv8_attn_workspace_bytes(const sixi_kv8_attn_params* p, size_t* bytes) {
    if (!bytes) return SIXI_E_INVALID_ARGUMENT;
    sixi::Kv8AttnArgs a;
    return resolve_attn(p, &a, bytes);
}

int sixi_kv8_attn(const sixi_kv8_attn_params* p) {
    sixi::Kv8AttnArgs a;
    size_t ws;
    const int rc = resolve_attn(p, &a, &ws);
    if (rc != SIXI_OK) return rc;
    if (!p->workspace) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(p->workspace, 256)) return SIXI_E_ALIGNMENT;
    if (p->workspace_bytes < ws) return SIXI_E_OUT_OF_BOUNDS;
    CacheViews cv{};
    (void)check_cache(p->cache, p->page_table != nullptr, &cv);
    const sixi_view* used[] = {&cv.k, &cv.v, &cv.ke, &cv.ve};
    for (const sixi_view* v : used)
        if (ranges_overlap(p->workspace, (int64_t)ws, v->data, view_span(*v, v->ne[0]))) return SIXI_E_INVALID_ARGUMENT;
    if (ranges_overlap(p->workspace, (int64_t)ws, p->q.data, view_span(p->q, a.D * elem_bytes(p->q.type))) ||
        ranges_overlap(p->workspace, (int64_t)ws, p->out.data, view_span(p->out, a.D * elem_bytes(p->out.type))) ||
        (a.mask && ranges_overlap(p->workspace, (int64_t)ws, p->mask.data, view_span(p->mask, p->mask.ne[0] * 2))) ||
        meets_arrays(p->workspace, (int64_t)ws, *p, a.S))
        return SIXI_E_INVALID_ARGUMENT;
    return sixi::launch_kv8_attn(a, static_cast<hipStream_t>(p->stream)) == hipSuccess ? SIXI_OK : SIXI_E_BACKEND;
}

}  // extern "C"
