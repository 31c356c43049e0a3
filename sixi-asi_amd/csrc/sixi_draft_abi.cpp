// sixi_draft_abi.cpp -- the C ABI of include/sixi_draft.h: validation on the host, the kernels in
// draft_verify.hip.
//
// As in sixi_attn_abi.cpp every error is a status (the reference's ErrorCode values of
// include/sixi_asi/common.hpp:40-67, negated).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "abi_util.hpp"
#include "device_util.hpp"
#include "draft_internal.hpp"
#include "sixi_draft.h"

namespace {

using namespace sixi_abi;

constexpr int64_t kMaxRows = sixi::kDraftMaxRows, kMaxDraftStreams = 65535, kMaxVocab = (int64_t)1 << 30;

int type_bytes(int32_t t) { return t == SIXI_TYPE_F32 ? 4 : t == SIXI_TYPE_F16 || t == SIXI_TYPE_BF16 ? 2 : 0; }

// Rows of V contiguous elements at any strides of whole elements.
int check_rows(const sixi_view& v, int64_t V, int64_t rows, int64_t S) {
    const int es = type_bytes(v.type);
    if (es == 0 || v.nb[0] != es) return SIXI_E_INVALID_ARGUMENT;
    if (v.ne[0] != V || v.ne[1] < rows || v.ne[2] != S || v.ne[3] != 1) return SIXI_E_INVALID_ARGUMENT;
    for (int d = 1; d < 3; ++d) {
        if (v.nb[d] < 0) return SIXI_E_INVALID_ARGUMENT;
        if (v.nb[d] % es) return SIXI_E_ALIGNMENT;
    }
    if (!aligned(v.data, es)) return SIXI_E_ALIGNMENT;
    int64_t span = 0;
    sixi_view w = v;
    w.nb[3] = 0;
    if (!mul_ok(V, es, &span) || view_span(w, span) < 0) return SIXI_E_INTEGER_OVERFLOW;
    return SIXI_OK;
}

int resolve(const sixi_draft_params* p, sixi::DraftArgs* out, size_t* ws) {
    if (!p || p->flags != 0) return SIXI_E_INVALID_ARGUMENT;
    const sixi_view& l = p->logits;
    const int64_t V = l.ne[0], rows = l.ne[1], S = l.ne[2];
    if (V <= 0 || rows <= 0 || S < 0 || (!l.data && S > 0)) return SIXI_E_INVALID_ARGUMENT;
    if (V > kMaxVocab || rows > kMaxRows || S > kMaxDraftStreams) return SIXI_E_UNSUPPORTED;
    int rc = check_rows(l, V, rows, S);
    if (rc != SIXI_OK) return rc;
    if (p->draft_probs.data && rows > 1) {
        rc = check_rows(p->draft_probs, V, rows - 1, S);
        if (rc != SIXI_OK) return rc;
    }
    if (rows > 1 && S > 0) {
        if (!p->draft || !p->u || p->draft_stride < 0 || p->u_stride < 0) return SIXI_E_INVALID_ARGUMENT;
        if (p->draft_stride > INT32_MAX || p->u_stride > INT32_MAX) return SIXI_E_INTEGER_OVERFLOW;
    }
    if (S > 0 && (!p->u_next || !p->keep || !p->token)) return SIXI_E_INVALID_ARGUMENT;
    for (const void* x : {(const void*)p->draft, (const void*)p->u, (const void*)p->u_next, (const void*)p->temperature,
                          (const void*)p->q_len, (const void*)p->keep, (const void*)p->token})
        if (!aligned(x, 4)) return SIXI_E_ALIGNMENT;
    // keep and token are written while the rest is read by other work-groups
    const int64_t l_bytes = view_span(l, V * type_bytes(l.type));
    for (const void* w : {(const void*)p->keep, (const void*)p->token}) {
        if (ranges_overlap(w, S * 4, l.data, l_bytes) || ranges_overlap(w, S * 4, p->u_next, S * 4) ||
            (p->temperature && ranges_overlap(w, S * 4, p->temperature, S * 4)) ||
            (p->q_len && ranges_overlap(w, S * 4, p->q_len, S * 4)) ||
            (p->draft_probs.data && rows > 1 &&
             ranges_overlap(w, S * 4, p->draft_probs.data, view_span(p->draft_probs, V * type_bytes(p->draft_probs.type)))) ||
            (rows > 1 && S > 0 && (ranges_overlap(w, S * 4, p->draft, ((S - 1) * p->draft_stride + rows - 1) * 4) ||
                                   ranges_overlap(w, S * 4, p->u, ((S - 1) * p->u_stride + rows - 1) * 4))))
            return SIXI_E_INVALID_ARGUMENT;
    }
    if (ranges_overlap(p->keep, S * 4, p->token, S * 4)) return SIXI_E_INVALID_ARGUMENT;

    sixi::DraftArgs a{};
    a.logits = static_cast<const char*>(l.data);
    a.l_nb1 = l.nb[1];
    a.l_nb2 = l.nb[2];
    a.l_type = l.type;
    if (rows > 1 && p->draft_probs.data) {
        a.probs = static_cast<const char*>(p->draft_probs.data);
        a.p_nb1 = p->draft_probs.nb[1];
        a.p_nb2 = p->draft_probs.nb[2];
        a.p_type = p->draft_probs.type;
    }
    a.draft = p->draft;
    a.draft_stride = p->draft_stride;
    a.u = p->u;
    a.u_stride = p->u_stride;
    a.u_next = p->u_next;
    a.temperature = p->temperature;
    a.q_len = p->q_len;
    a.keep = p->keep;
    a.token = p->token;
    a.V = (int32_t)V;
    a.n_rows = (int32_t)rows;
    a.S = (int32_t)S;
    a.chunks = (int32_t)((V + sixi::kDraftChunk - 1) / sixi::kDraftChunk);
    // four chunks in a row where one each would be more than four work-groups for each of 8 places of a CU
    a.run = S * rows * a.chunks > 4 * 8 * (int64_t)sixi::device_cu_count() ? 4 : 1;
    a.n_parts = (a.chunks + a.run - 1) / a.run;
    // a work-group of the draw first forms the accept chain again: no more of them than run at once, 3 on a CU
    // (32 streams of 61 chunks: 25 us, with a chunk each 29)
    const int64_t places = 3 * (int64_t)sixi::device_cu_count();
    a.draw_run = (int32_t)std::clamp<int64_t>((S * a.chunks + places - 1) / places, 1, 8);
    const int64_t parts = S * rows * a.n_parts * (int64_t)sizeof(sixi::DraftPart);  // < 2^16 * 2^10 * 2^18 * 2^4
    const int64_t draws = S * a.chunks * (int64_t)sizeof(sixi::DraftDraw);
    *ws = (size_t)(parts + draws) + (size_t)S * sizeof(int32_t);
    *ws = (*ws + 255) / 256 * 256;
    if (*ws == 0) *ws = 256;
    a.parts = static_cast<sixi::DraftPart*>(p->workspace);
    if (p->workspace) {
        a.draws = reinterpret_cast<sixi::DraftDraw*>(static_cast<char*>(p->workspace) + parts);
        a.counts = reinterpret_cast<int32_t*>(static_cast<char*>(p->workspace) + parts + draws);
    }
    *out = a;
    return SIXI_OK;
}

}  // namespace

extern "C" {

int sixi_draft_validate(const sixi_draft_params* p) {
    sixi::DraftArgs a;
    size_t ws;
    return resolve(p, &a, &ws);
}

int sixi_draft_workspace_bytes(const sixi_draft_params* p, size_t* bytes) {
    if (!bytes) return SIXI_E_INVALID_ARGUMENT;
    sixi::DraftArgs a;
    return resolve(p, &a, bytes);
}

int sixi_draft_verify(const sixi_draft_params* p) {
    sixi::DraftArgs a;
    size_t ws;
    const int rc = resolve(p, &a, &ws);
    if (rc != SIXI_OK) return rc;
    if (a.S == 0) return SIXI_OK;
    if (!p->workspace) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(p->workspace, 256)) return SIXI_E_ALIGNMENT;
    if (p->workspace_bytes < ws) return SIXI_E_OUT_OF_BOUNDS;
    const int64_t l_bytes = view_span(p->logits, p->logits.ne[0] * type_bytes(p->logits.type));
    if (ranges_overlap(p->workspace, (int64_t)ws, p->logits.data, l_bytes) ||
        ranges_overlap(p->workspace, (int64_t)ws, p->keep, a.S * 4) || ranges_overlap(p->workspace, (int64_t)ws, p->token, a.S * 4) ||
        (a.probs && ranges_overlap(p->workspace, (int64_t)ws, a.probs,
                                   view_span(p->draft_probs, p->draft_probs.ne[0] * type_bytes(a.p_type)))))
        return SIXI_E_INVALID_ARGUMENT;
    for (const void* r : {(const void*)p->u_next, (const void*)p->temperature, (const void*)p->q_len})
        if (r && ranges_overlap(p->workspace, (int64_t)ws, r, a.S * 4)) return SIXI_E_INVALID_ARGUMENT;
    if (a.n_rows > 1 && (ranges_overlap(p->workspace, (int64_t)ws, a.draft, ((a.S - 1) * a.draft_stride + a.n_rows - 1) * 4) ||
                         ranges_overlap(p->workspace, (int64_t)ws, a.u, ((a.S - 1) * a.u_stride + a.n_rows - 1) * 4)))
        return SIXI_E_INVALID_ARGUMENT;
    return sixi::launch_draft_verify(a, static_cast<hipStream_t>(p->stream)) == hipSuccess ? SIXI_OK : SIXI_E_BACKEND;
}

}  // extern "C"
