// rope_internal.hpp -- kernel arguments shared by the rotary ABI (sixi_rope_abi.cpp) and its kernel
// (rope.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sixi {

// One tensor's rows.  Byte strides: head, row, stream.
struct RopeTensor {
    const char* in;
    char* out;
    int64_t i_nb1, i_nb2, i_nb3, o_nb1, o_nb2, o_nb3;
    const float* norm;
    int32_t in_f16, out_f16, heads;
};

struct RopeArgs {
    RopeTensor t[2];  // Q, K (heads 0: none)
    const double* freqs;
    const int32_t* kv_len;
    const int32_t* pos;
    int64_t pos_stride;
    const int32_t* q_len;
    float eps, mscale;
    int32_t n_rot, interleaved, inverse, D, n_rows, S;
};

hipError_t launch_qk_rope(const RopeArgs& a, hipStream_t stream);

}  // namespace sixi
