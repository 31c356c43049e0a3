// kv8_internal.hpp -- kernel arguments shared by the 8-bit cache's ABI (sixi_kv8_abi.cpp) and its
// kernels (kv8_store.hip, kv8_attn.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sixi_kv8.h"

namespace sixi {

constexpr int kBlk = SIXI_KV8_BLOCK_CELLS;
constexpr int kPageBlocks = SIXI_KV_PAGE_CELLS / SIXI_KV8_BLOCK_CELLS;

// One tensor's codes and exponents (strides in bytes: block, head, stream or page).
struct Kv8Tensor {
    char* codes;
    int8_t* exps;
    int64_t nb[3];
    int64_t e_nb[3];
};

// Where a stream's blocks lie.  pt null: block b of stream s at b * nb[0] + s * nb[2].
struct Kv8Pages {
    const int32_t* pt;
    int64_t pt_stride;
    int32_t n_pages;
    int32_t n_blocks;  // blocks of a stream (paged: of its whole table row)
};

// Rows of both tensors against cells kv_len[s] + j.  Byte strides of the rows: row, head, stream.
struct Kv8RowsArgs {
    char* rows[2];
    int64_t r_nb1[2], r_nb2[2], r_nb3[2];
    int32_t f16[2];
    Kv8Tensor t[2];
    Kv8Pages pages;
    const int32_t* kv_len;
    const int32_t* q_len;
    int32_t D, n_rows, Hkv, S;
};

hipError_t launch_kv8_write(const Kv8RowsArgs& a, hipStream_t stream);
hipError_t launch_kv8_read(const Kv8RowsArgs& a, hipStream_t stream);

// Where the pieces of a stream's cells begin.
struct Kv8Place {
    int32_t s, tiles, pieces, at;  // stream, its tiles, pieces of each, number of its first piece
};

struct Kv8AttnArgs {
    const char* q;
    int64_t q_nb1, q_nb2, q_nb3;  // row, head, stream
    int32_t q_f16;
    char* out;
    int64_t o_nb1, o_nb2, o_nb3;  // head, row, stream
    int32_t o_f16;
    Kv8Tensor k, v;
    Kv8Pages pages;
    const int32_t* kv_len;
    const int32_t* q_len;
    const char* mask;             // EXPLICIT: f16 rows
    int64_t m_nb1, m_nb3;         // row, stream (0: one for all)
    int32_t mode;
    int32_t S, H, Hkv, G, n_q, n_kv, D;
    float scale_log2;             // |scale| * log2(e); the sign goes into Q
    float q_sign;
    float* part;                  // workspace: partial results of the pieces
    Kv8Place* places;             // and, behind them, each stream's place
    int32_t waves;                // row tiles of 32 that a work-group takes (1: its waves share the cells)
    int32_t target;               // work-groups that the cells are cut for
    int32_t least;                // blocks of a piece at least
    int32_t grid;                 // pieces at most
    int32_t cut;                  // whether cells may be cut (partial results in the workspace)
    int64_t code_bytes;           // codes of all cells that a call may see
    int32_t once;                 // codes are read past the caches
};

hipError_t launch_kv8_attn(const Kv8AttnArgs& a, hipStream_t stream);

// Chooses waves, target, least and grid for the shape; the workspace's bytes.
size_t kv8_attn_plan(Kv8AttnArgs& a);

}  // namespace sixi
