// sample.h — the draw of next tokens (sample.hip), for decode.hip too.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "../../include/welvet_hip.h"

namespace wv {

struct SampleArgs {
    const float* logits;
    int64_t stride;
    int rows, vocab;
    wv_sampling p;       // per-row arrays, each may be null
    int32_t* tokens;     // [rows], may be null with state
    float* probs;        // [rows] or null
    // A decode step's state {pos, token, next, step}: the draw of its one row
    // reads uniform[step], records the token as generated token `step` and
    // moves the state on, as k_argmax_advance does.
    int32_t* state;
    int32_t* gen;
    int gen_cap, advance;
};
// Rows of many logits are cut into slices where the caller gives scratch
// (sample_scratch_floats, 16-byte aligned; 0: none is used).
size_t sample_scratch_floats(int rows, int vocab);
int launch_sample(const SampleArgs& a, hipStream_t s, float* scratch = nullptr);

}  // namespace wv
