// draft_internal.hpp -- kernel arguments shared by the draft verification's ABI (sixi_draft_abi.cpp) and
// its kernels (draft_verify.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sixi {

constexpr int kDraftChunk = 4096;  // logits of a row that one work-group takes
constexpr int kDraftMaxRows = 1024;

// Some chunks of a row: the largest logit, the lowest token that has it, and the sum of exp((l - max) / T).
struct DraftPart {
    double sum;
    float top;
    int32_t at;
};
// A chunk of the row that the next token is drawn from: weights of the draw and of p, the last token with
// a weight in each.
struct DraftDraw {
    double w, p;
    int32_t last_w, last_p;
};

// What a stream's rows come to.
struct DraftVerdict {
    double inv_z;   // 1 / the sum of the weights of the row below
    double c;       // log2(e) / temperature; 0: greedy
    int32_t row;    // the row that the next token is drawn from
    int32_t d;      // its drafted token (V: none in range); -1 behind the last one
    float top;      // its largest logit
    int32_t at;     // the lowest token that has it (greedy streams)
};

struct DraftArgs {
    const char* logits;
    int64_t l_nb1, l_nb2;  // row, stream
    const char* probs;     // may be null
    int64_t p_nb1, p_nb2;
    int32_t l_type, p_type;
    const int32_t* draft;
    int64_t draft_stride;
    const float* u;
    int64_t u_stride;
    const float* u_next;
    const float* temperature;
    const int32_t* q_len;
    int32_t* keep;
    int32_t* token;
    DraftPart* parts;  // [S][n_rows][n_parts]
    DraftDraw* draws;  // [S][chunks]
    int32_t* counts;   // [S]: chunks whose share is in draws
    int32_t V, n_rows, S, chunks;  // chunks of a row
    int32_t run, n_parts;          // chunks that a work-group of the rows takes; such work-groups of a row
    int32_t draw_run;              // chunks that a work-group of the draw takes
};

hipError_t launch_draft_verify(const DraftArgs& a, hipStream_t stream);

}  // namespace sixi
