// sixi_rope_abi.cpp -- the C ABI of include/sixi_rope.h: validation and the frequency table on the host,
// the kernel in rope.hip.
//
// As in sixi_attn_abi.cpp every error is a status (the reference's ErrorCode values of
// include/sixi_asi/common.hpp:40-67, negated).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "abi_util.hpp"
#include "rope_internal.hpp"
#include "sixi_rope.h"

namespace {

using namespace sixi_abi;

bool same_view(const sixi_view& a, const sixi_view& b) {
    if (a.data != b.data || a.type != b.type) return false;
    for (int i = 1; i < 4; ++i)
        if (a.ne[i] > 1 && a.nb[i] != b.nb[i]) return false;
    return true;
}

int check_view(const sixi_view& v) {
    if (elem_bytes(v.type) == 0) return SIXI_E_INVALID_ARGUMENT;
    for (int i = 0; i < 4; ++i)
        if (v.ne[i] < 0 || v.nb[i] < 0) return SIXI_E_INVALID_ARGUMENT;
    if (!v.data && v.ne[0] > 0 && v.ne[1] > 0 && v.ne[2] > 0 && v.ne[3] > 0) return SIXI_E_INVALID_ARGUMENT;
    if (v.nb[0] != elem_bytes(v.type)) return SIXI_E_INVALID_ARGUMENT;
    for (int i = 1; i < 4; ++i)
        if (v.ne[i] > INT32_MAX) return SIXI_E_INTEGER_OVERFLOW;
    if (view_span(v, v.ne[0] * elem_bytes(v.type)) < 0) return SIXI_E_INTEGER_OVERFLOW;
    if (!aligned(v.data, 16) || v.nb[1] % 16 || v.nb[2] % 16 || v.nb[3] % 16) return SIXI_E_ALIGNMENT;
    return SIXI_OK;
}

// A tensor and where its rotation goes.
int check_pair(const sixi_view& in, const sixi_view& out, sixi::RopeTensor* t) {
    int rc = check_view(in);
    if (rc == SIXI_OK) rc = check_view(out);
    if (rc != SIXI_OK) return rc;
    for (int i = 0; i < 4; ++i)
        if (in.ne[i] != out.ne[i]) return SIXI_E_INVALID_ARGUMENT;
    const int64_t ib = in.ne[0] * elem_bytes(in.type), ob = out.ne[0] * elem_bytes(out.type);
    if (view_span(out, ob) > 0 && !rows_disjoint(out, ob)) return SIXI_E_INVALID_ARGUMENT;
    // in place, row for row, or apart: a row is read by the lanes that write it, and by no others
    if (!same_view(in, out) && views_overlap(in, ib, out, ob)) return SIXI_E_INVALID_ARGUMENT;
    t->in = static_cast<const char*>(in.data);
    t->out = static_cast<char*>(const_cast<void*>(out.data));
    t->i_nb1 = in.nb[1];
    t->i_nb2 = in.nb[2];
    t->i_nb3 = in.nb[3];
    t->o_nb1 = out.nb[1];
    t->o_nb2 = out.nb[2];
    t->o_nb3 = out.nb[3];
    t->in_f16 = in.type == SIXI_TYPE_F16;
    t->out_f16 = out.type == SIXI_TYPE_F16;
    t->heads = (int32_t)in.ne[1];
    return SIXI_OK;
}

int resolve(const sixi_qk_rope_params* p, sixi::RopeArgs* out) {
    if (!p || (p->flags & ~SIXI_ROPE_INVERSE) != 0) return SIXI_E_INVALID_ARGUMENT;
    if (p->layout != SIXI_ROPE_HALF && p->layout != SIXI_ROPE_INTERLEAVED) return SIXI_E_INVALID_ARGUMENT;
    sixi::RopeArgs a{};
    int rc = check_pair(p->q, p->q_out, &a.t[0]);
    if (rc != SIXI_OK) return rc;
    const int64_t D = p->q.ne[0], n_rows = p->q.ne[2], S = p->q.ne[3];
    const bool has_k = p->k.data != nullptr;
    if (has_k) {
        rc = check_pair(p->k, p->k_out, &a.t[1]);
        if (rc != SIXI_OK) return rc;
        if (p->k.ne[0] != D || p->k.ne[2] != n_rows || p->k.ne[3] != S) return SIXI_E_INVALID_ARGUMENT;
        // no output may be what another work-group reads or writes
        auto bytes = [](const sixi_view& v) { return v.ne[0] * elem_bytes(v.type); };
        if (views_overlap(p->q_out, bytes(p->q_out), p->k, bytes(p->k)) || views_overlap(p->k_out, bytes(p->k_out), p->q, bytes(p->q)) ||
            views_overlap(p->q_out, bytes(p->q_out), p->k_out, bytes(p->k_out)))
            return SIXI_E_INVALID_ARGUMENT;
    }
    if (D <= 0 || D % 16 != 0 || D > 256) return SIXI_E_UNSUPPORTED;
    if (S > 65535 || n_rows > (1 << 23) || p->q.ne[1] > 65535 || (has_k && p->k.ne[1] > 65535)) return SIXI_E_UNSUPPORTED;
    if (p->n_rot < 0 || p->n_rot > D || p->n_rot % 16 != 0) return SIXI_E_INVALID_ARGUMENT;
    if (p->n_rot > 0 && !p->freqs) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(p->freqs, 8) || !aligned(p->kv_len, 4) || !aligned(p->pos, 4) || !aligned(p->q_len, 4)) return SIXI_E_ALIGNMENT;
    const bool norm = p->q_norm != nullptr;
    if (has_k ? (p->k_norm != nullptr) != norm : p->k_norm != nullptr) return SIXI_E_INVALID_ARGUMENT;
    if (norm && (p->flags & SIXI_ROPE_INVERSE)) return SIXI_E_INVALID_ARGUMENT;
    if (norm && (!std::isfinite(p->eps) || p->eps < 0.0f)) return SIXI_E_INVALID_ARGUMENT;
    if (!aligned(p->q_norm, 16) || !aligned(p->k_norm, 16)) return SIXI_E_ALIGNMENT;
    if (!std::isfinite(p->mscale)) return SIXI_E_INVALID_ARGUMENT;
    if (p->pos && p->pos_stride < 0) return SIXI_E_INVALID_ARGUMENT;
    if (p->pos && p->pos_stride > INT32_MAX) return SIXI_E_INTEGER_OVERFLOW;
    // rows are written while other work-groups read these
    const struct { const void* p; int64_t bytes; } read[] = {
        {p->freqs, (int64_t)p->n_rot / 2 * 8},  {p->q_norm, norm ? D * 4 : 0}, {p->k_norm, p->k_norm ? D * 4 : 0},
        {p->kv_len, p->kv_len ? S * 4 : 0},     {p->q_len, p->q_len ? S * 4 : 0},
        {p->pos, p->pos && S > 0 ? ((S - 1) * p->pos_stride + n_rows) * 4 : 0}};
    for (int i = 0; i < (has_k ? 2 : 1); ++i) {
        const sixi_view& w = i ? p->k_out : p->q_out;
        const int64_t span = view_span(w, D * elem_bytes(w.type));
        for (const auto& r : read)
            if (ranges_overlap(w.data, span, r.p, r.bytes)) return SIXI_E_INVALID_ARGUMENT;
    }
    a.t[0].norm = p->q_norm;
    a.t[1].norm = p->k_norm;
    a.freqs = p->freqs;
    a.kv_len = p->kv_len;
    a.pos = p->pos;
    a.pos_stride = p->pos_stride;
    a.q_len = p->q_len;
    a.eps = p->eps;
    a.mscale = p->mscale;
    a.n_rot = p->n_rot;
    a.interleaved = p->layout == SIXI_ROPE_INTERLEAVED;
    a.inverse = (p->flags & SIXI_ROPE_INVERSE) != 0;
    a.D = (int32_t)D;
    a.n_rows = (int32_t)n_rows;
    a.S = (int32_t)S;
    *out = a;
    return SIXI_OK;
}

}  // namespace

extern "C" {

int sixi_rope_frequencies(int32_t n_rot, double base, const sixi_rope_scaling* sc, double* freqs, float* mscale) {
    if (n_rot < 0 || n_rot % 2 != 0 || !freqs || !mscale) return SIXI_E_INVALID_ARGUMENT;
    if (!std::isfinite(base) || base <= 1.0) return SIXI_E_INVALID_ARGUMENT;
    const int32_t kind = sc ? sc->kind : SIXI_ROPE_SCALE_NONE;
    if (kind < SIXI_ROPE_SCALE_NONE || kind > SIXI_ROPE_SCALE_YARN) return SIXI_E_INVALID_ARGUMENT;
    const double factor = kind == SIXI_ROPE_SCALE_NONE ? 1.0 : sc->factor;
    if (!std::isfinite(factor) || factor < 1.0) return SIXI_E_INVALID_ARGUMENT;
    double lo = 0.0, hi = 0.0;
    if (kind == SIXI_ROPE_SCALE_YARN) {
        if (sc->trained_len <= 0 || !(sc->beta_slow > 0.0) || !(sc->beta_fast > sc->beta_slow) || !std::isfinite(sc->beta_fast))
            return SIXI_E_INVALID_ARGUMENT;
        // the pair that makes `turns` turns over the trained positions
        auto pair = [&](double turns) { return n_rot * std::log(sc->trained_len / (turns * 2.0 * M_PI)) / (2.0 * std::log(base)); };
        lo = std::fmax(0.0, std::floor(pair(sc->beta_fast)));
        hi = std::fmin((double)n_rot - 1.0, std::ceil(pair(sc->beta_slow)));
    }
    for (int32_t i = 0; i < n_rot / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / n_rot);
        double stretch = kind == SIXI_ROPE_SCALE_LINEAR ? 1.0 : 0.0;  // the share of f / factor
        if (kind == SIXI_ROPE_SCALE_YARN) stretch = std::fmin(1.0, std::fmax(0.0, (i - lo) / std::fmax(hi - lo, 1e-3)));
        freqs[i] = f / factor * stretch + f * (1.0 - stretch);
    }
    *mscale = kind == SIXI_ROPE_SCALE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
    return SIXI_OK;
}

int sixi_qk_rope_validate(const sixi_qk_rope_params* p) {
    sixi::RopeArgs a;
    return resolve(p, &a);
}

int sixi_qk_rope(const sixi_qk_rope_params* p) {
    sixi::RopeArgs a;
    const int rc = resolve(p, &a);
    if (rc != SIXI_OK) return rc;
    return sixi::launch_qk_rope(a, static_cast<hipStream_t>(p->stream)) == hipSuccess ? SIXI_OK : SIXI_E_BACKEND;
}

}  // extern "C"
