/*
 * sixi_rope.h -- C ABI of rotary positions for Q and K (gfx950): half and interleaved pairs, a part
 * of the head, any frequencies (scaled for long contexts), with an optional RMS norm in front.
 *
 * sixi_qk_prologue (sixi_layer.h) serves one model's layer and caches of ggml types: the half layout,
 * angles by repeated f32 products as ggml forms them.  This call is for the rest: caches that are
 * written by a call of their own (sixi_kv8.h), scaled contexts, trees of drafted tokens (positions
 * that do not follow the rows), and positions where an f32 angle is off by more than the rotation
 * can bear (at position 180000 by up to 8e-3 radians).  Ownership and threading as in sixi_attn.h.
 */
#ifndef SIXI_ROPE_H
#define SIXI_ROPE_H

#include "sixi_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    SIXI_ROPE_HALF = 0,         /* pairs (i, i + n_rot/2)                                        */
    SIXI_ROPE_INTERLEAVED = 1   /* pairs (2i, 2i + 1)                                            */
};

/* sixi_qk_rope_params.flags: turn by the negative angle (undoes a rotation, up to mscale^2; the
 * product with the rotation's transpose).  Not with norm weights. */
enum { SIXI_ROPE_INVERSE = 1 };

enum {
    SIXI_ROPE_SCALE_NONE = 0,
    SIXI_ROPE_SCALE_LINEAR = 1, /* every frequency / factor                                      */
    SIXI_ROPE_SCALE_YARN = 2    /* slow pairs / factor, fast ones as trained, a ramp between     */
};

typedef struct sixi_rope_scaling {
    int32_t kind;           /* SIXI_ROPE_SCALE_*                                                 */
    int32_t trained_len;    /* YARN: positions the model was trained on                          */
    double factor;          /* >= 1                                                              */
    double beta_fast;       /* YARN: turns over trained_len above which a pair is left (32)      */
    double beta_slow;       /* YARN: turns below which a pair is stretched by factor (1)         */
} sixi_rope_scaling;

/* Host: the n_rot/2 frequencies (radians per position) base^(-2i/n_rot), scaled, and the factor on
 * the rotated values (*mscale; 1, or 0.1 ln(factor) + 1 with YARN).  scaling may be NULL. */
int sixi_rope_frequencies(int32_t n_rot, double base, const sixi_rope_scaling* scaling, double* freqs, float* mscale);

typedef struct sixi_qk_rope_params {
    sixi_view q;            /* [D, H, n_rows, S] f32 or f16, rows contiguous                     */
    sixi_view k;            /* [D, Hkv, n_rows, S], or data NULL: no K                           */
    sixi_view q_out;        /* the shape of q, f32 or f16; may be q itself (same strides, type)  */
    sixi_view k_out;
    const double* freqs;    /* device [n_rot / 2]: radians per position                          */
    const float* q_norm;    /* device [D], or NULL: no norm (both or none where there is a K)    */
    const float* k_norm;
    float eps;              /* of the norm                                                       */
    float mscale;           /* factor on the rotated values                                      */
    int32_t n_rot;          /* rotated dims, the first of the head: a multiple of 16, at most D  */
    int32_t layout;         /* SIXI_ROPE_HALF or SIXI_ROPE_INTERLEAVED                           */
    int32_t flags;          /* 0 or SIXI_ROPE_INVERSE                                            */
    int32_t reserved;
    const int32_t* kv_len;  /* device [S]: position of row 0, or NULL (0)                        */
    const int32_t* pos;     /* device: position of row j of stream s at pos[s * pos_stride + j]
                               (kv_len is not read then), or NULL                                */
    int64_t pos_stride;
    const int32_t* q_len;   /* device [S]: rows of stream s (<= n_rows), or NULL (= n_rows)      */
    void* stream;
} sixi_qk_rope_params;

/* For every row j < q_len[s], head and pair i of the first n_rot dims, with a = position * freqs[i]:
 *   (x0, x1) -> mscale * (x0 cos a - x1 sin a, x1 cos a + x0 sin a)
 * after x = x / sqrt(mean(x^2) + eps) * norm where norm weights are given.  Dims past n_rot pass
 * (normed, unscaled).  Angles are reduced in 64 bits.  D is a multiple of 16 up to 256; rows, weights
 * and strides 16-byte aligned.  Rows past q_len are not written.  At most 2^23 rows of a stream and
 * 65535 heads and streams. */
int sixi_qk_rope(const sixi_qk_rope_params* p);

/* Host-side validation only: SIXI_OK or the error sixi_qk_rope returns. */
int sixi_qk_rope_validate(const sixi_qk_rope_params* p);

#ifdef __cplusplus
}
#endif
#endif /* SIXI_ROPE_H */
