/*
 * sixi_kv8.h -- C ABI of a KV cache held in 8 bits (gfx950): int8 codes with one power-of-two
 * scale for each block of 32 cells and kv-head, the store and read-back of its rows, and the
 * attention that reads it.
 *
 * A value is code * 2^e, code in [-127, 127] and e in [SIXI_KV8_EXP_MIN, SIXI_KV8_EXP_MAX], with K
 * and V each their own e per (block, head).  A cell takes D + 1/32 bytes per head and tensor: about
 * half of f16, and 6 % less than q8_0.  Powers of two make the conversions exact: a code is the
 * value's nearest multiple of 2^e (ties to even), whatever computes it, and the attention applies
 * the scales to sums and exponents without a rounding.
 *
 * Layout.  A block of 32 cells of one head is contiguous, 32 * D bytes:
 *   K  [D / 16][32 cells][16 dims]      V  [D][32 cells]
 * i.e. in the order in which the matrix cores take them, so that 64 lanes load 1 KiB in one piece
 * and nothing is transposed on the way.  Blocks, heads and streams (or pages) lie at any strides of
 * 16 bytes.  Applications reach the values through sixi_kv8_write and sixi_kv8_read; whole blocks
 * (with their exponents) may be copied as bytes.
 *
 * Cells, lengths and pages are those of sixi_attn.h and sixi_kv.h: row j of stream s sits in cell
 * kv_len[s] + j; a page holds 256 cells (8 blocks).  Rolling back shortens kv_len and moves nothing.
 *
 * The reference has caches of whole ggml types only (src/core/core_execution.cpp:2600-2608,
 * --kv-type): no counterpart there.  Ownership and threading as in sixi_attn.h.
 */
#ifndef SIXI_KV8_H
#define SIXI_KV8_H

#include "sixi_attn.h"
#include "sixi_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define SIXI_KV8_BLOCK_CELLS 32
#define SIXI_KV8_EXP_MIN (-40)
#define SIXI_KV8_EXP_MAX 40

/* K and V of one layer.  Strides are bytes, of a block, a head and a stream (paged: a page); the
 * blocks of the codes and of the exponents must not overlap one another. */
typedef struct sixi_kv8_cache {
    void* k;                /* int8 codes, 16-byte aligned                                       */
    void* v;
    int8_t* k_exp;          /* exponents; entries outside the range count as its nearest end     */
    int8_t* v_exp;
    int64_t k_nb[3];        /* block, head, stream: multiples of 16                              */
    int64_t v_nb[3];
    int64_t k_exp_nb[3];    /* block, head, stream                                               */
    int64_t v_exp_nb[3];
    int32_t head_dim;       /* D: 128 or 256                                                     */
    int32_t n_heads;        /* kv-heads                                                          */
    int64_t n_blocks;       /* blocks of a stream; paged: 8 (SIXI_KV_PAGE_CELLS / 32)            */
    int64_t n;              /* streams; paged: pages                                             */
} sixi_kv8_cache;

typedef struct sixi_kv8_rows_params {
    sixi_view k;            /* [D, n_rows, Hkv, S] f32 or f16, rows contiguous and 16-byte       */
    sixi_view v;            /* aligned: read by sixi_kv8_write, written by sixi_kv8_read         */
    sixi_kv8_cache cache;
    const int32_t* kv_len;  /* device [S]: cell of row 0, or NULL (cell 0)                       */
    const int32_t* q_len;   /* device [S]: rows of stream s (<= n_rows), or NULL (= n_rows)      */
    int32_t flags;          /* reserved, must be 0                                               */
    int32_t reserved;
    void* stream;           /* hipStream_t; NULL = the null stream                               */
    /* Paged cache (optional, as sixi_attn_params): block b of stream s is block b % 8 of page
     * page_table[s * page_table_stride + b / 8]; entries are clamped to [0, n). */
    const int32_t* page_table;
    int64_t page_table_stride;
} sixi_kv8_rows_params;

/* Stores row j < q_len[s] of stream s in cell kv_len[s] + j, K and V of every head in one launch.
 * Rows whose cell falls outside the cache are not stored.  For each block that receives rows:
 *   - its cells before the first row stored are kept, cells behind the last row hold nothing;
 *   - e is the smallest exponent in range with max |x| <= 127 * 2^e over the finite values of the
 *     new rows, and not less than the block's own if it keeps cells;
 *   - the kept cells' codes become the nearest multiples of the new scale (ties to even): a
 *     scale grows as louder rows arrive, and starts anew when a block is written from its first
 *     cell.  The bytes of cells behind the last row do not change.
 * Infinities are stored as +-127 * 2^e, NaN as 0.  A block is written whole: streams that share a
 * page must not store into the same block of it in one call, nor in calls that may overlap. */
int sixi_kv8_write(const sixi_kv8_rows_params* p);

/* Reads cell kv_len[s] + j into row j < q_len[s] of k and v.  Exact in f32; f16 rows hold the
 * nearest f16 (the value itself for exponents -24 .. 8), at most 65504 in size.  Rows whose cell
 * falls outside the cache, and rows past q_len, are not written. */
int sixi_kv8_read(const sixi_kv8_rows_params* p);

/* Host-side validation only: SIXI_OK or the error that sixi_kv8_write (read = 0) or
 * sixi_kv8_read (read != 0) returns. */
int sixi_kv8_rows_validate(const sixi_kv8_rows_params* p, int read);

/* Registers a page pool in this format (n = the pool's pages, n_blocks = 8) whose pages
 * copy-on-write duplicates, codes and exponents (sixi_kv_pool_attach for the other formats).  The
 * blocks of a page must lie at the head's start, one after the other, in all four tensors. */
int sixi_kv8_pool_attach(sixi_kv_pool* pool, const sixi_kv8_cache* pages);

typedef struct sixi_kv8_attn_params {
    sixi_view q;            /* [D, n_q, H, S] f16 or f32 (rounded to f16 as it is read), rows
                               contiguous and 16-byte aligned                                    */
    sixi_kv8_cache cache;
    sixi_view out;          /* [D, H, n_q, S] f32 or f16, rows contiguous and 16-byte aligned    */
    const int32_t* kv_len;  /* device [S]: cells cached before the block, or NULL                */
    const int32_t* q_len;   /* device [S]: rows of stream s (<= n_q), or NULL (= n_q)            */
    int32_t mask_mode;      /* SIXI_MASK_*, as sixi_attn_params                                  */
    int32_t flags;          /* reserved, must be 0                                               */
    sixi_view mask;         /* EXPLICIT only: f16 [n_kv, >= n_q, 1, 1 or S], 2-byte aligned      */
    float scale;            /* finite                                                            */
    float reserved_f;
    void* workspace;        /* device scratch of >= sixi_kv8_attn_workspace_bytes() bytes,
                               256-byte aligned, no initialisation                               */
    size_t workspace_bytes;
    void* stream;
    const int32_t* page_table;  /* as above                                                      */
    int64_t page_table_stride;
} sixi_kv8_attn_params;

/* O = softmax(scale * Q K^T + mask) V over the 8-bit cache, for every stream, head and row j <
 * q_len[s]: decode, verify and prefill by the row count.  q-heads g*G .. g*G+G-1 share kv-head g
 * (G = H / Hkv, any ratio).  The cells a row sees are those of sixi_attn_params.mask_mode; kv_len[s]
 * is clamped to [0, n_kv - q_len[s]] on the device.  A row that sees no cell is zero; rows
 * j >= q_len[s] are not written.  Q K^T and the sums run in f32 over exact products of the codes and
 * Q in f16 (an f32 Q is rounded to f16 as it is read); the softmax's weights are rounded to f16 in
 * front of the product with V.  At most 2^23 tiles of 32 rows (n_q * G of a head) in a call. */
int sixi_kv8_attn(const sixi_kv8_attn_params* p);

/* Workspace the call needs for this description (not dependent on the device-side lengths). */
int sixi_kv8_attn_workspace_bytes(const sixi_kv8_attn_params* p, size_t* bytes);

/* Host-side validation only: SIXI_OK or the error sixi_kv8_attn returns, apart from the workspace's. */
int sixi_kv8_attn_validate(const sixi_kv8_attn_params* p);

#ifdef __cplusplus
}
#endif
#endif /* SIXI_KV8_H */
